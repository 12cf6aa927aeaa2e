// Expanded attention of a latent cache's prompts:
//
//   out_ht = sum_j p_j v_hj / sum_j p_j,
//   p_j = exp(scale (q_ht[:128] . k_hj + q_ht[128:] . r_j) - m),
//
// j over the keys that row t sees, r_j the rotated part of key j that every head
// shares.
//
// Work split.  128 rows (64 where there are no more) of a (sequence, head) form a
// unit, its keys up to the last that one of them sees are tiles of 32.  A fixed grid
// takes equal ranges of the flat list of all units' tiles (and of what units cost
// beside them); units that cross ranges leave partials (maximum, sum, output), which
// expanded_merge_kernel joins.  A head's units lie near each other in the list, and an
// XCD has ranges that do, so that row blocks that read the same keys at about the same
// time find them in its L2: of 21 million cache lines of the case below 9 are read past
// it, with row blocks apart 20.
//
// Matrix form.  As in the absorbed form: S^T = K Q^T, O^T += V^T P^T, a lane holding
// keys of one query row, a wavefront 16 rows.  fp32 numbers are sums of 16-bit terms,
// split once a workgroup on their way into LDS.
// - expanded_kernel: two fp16 terms (22 bits and a sign: the rounding of an fp32
//   number), of whose four products the three above 2^-22 of the largest are taken.
//   fp16's range asks for powers of two: a query row's own, one for the keys and one
//   for the values of a unit's part, by the largest numbers of its first eight keys
//   that all its rows see.  Those keys go to [2^4, 2^5) and values to [2^8, 2^9), so
//   that keys 2^11 and values 2^7 times as large fit; 2^-25 is lost of numbers as
//   scaled.  Probabilities carry a factor of 2^8.
// - expanded_redo_kernel: three bf16 terms (24 bits, fp32's range), of whose nine
//   products the six above 2^-26 are taken.  It computes parts again whose unit the
//   first one marked: with numbers past its range, a sum or output that is not finite
//   (what a row does not see can show that way), or rows of which the 2^-25 might
//   count, by the size of their scores or outputs.
//
// What bounds it: 4 x 32 heads, 512 rows over 4096 keys are 161 Gflop, three times
// that in products of terms: 413 us at the rate of a large fp16 matrix product, 543 to
// 558 here (1300 to 1450 where parts are computed again).  Of a step's 4300 cycles a SIMD's
// matrix instructions take 2080, its other vector instructions 1300; the two of its
// wavefronts take turns, and what is left are the waits of one for the other at the
// step's two barriers and the scalar work between tiles.  Steps on the way: three bf16
// terms and six products throughout 936 us; two fp16 terms 653; eight wavefronts of 16
// rows, two a SIMD, for four of 32: 634; four of them half a step behind 610; tiles by
// scalar bases 584; heads woven 543.
#include "bf16.hpp"
#include "latent.hpp"
#include "latent_detail.hpp"
#include "prefill_bmma.hpp"

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <type_traits>

namespace helix::hip {
namespace {

using latent_detail::align256;
using latent_detail::clamped_count;
using latent_detail::divide;
using latent_detail::kNoWeights;
using latent_detail::lane_scan;
using latent_detail::matrix_step;
using latent_detail::part_sum;
using latent_detail::row_factor;
using latent_detail::uniform_long;
using latent_detail::v4u;
using prefill_detail::exp2_ratio;
using prefill_detail::row_max;
using prefill_detail::row_sum;
using prefill_detail::uniform_read;
using prefill_detail::v4f;
using prefill_detail::v4s;

typedef unsigned v2u __attribute__((ext_vector_type(2)));
typedef float v2f __attribute__((ext_vector_type(2)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef __bf16 v2bf __attribute__((ext_vector_type(2)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kKeyDim = static_cast<int>(kLatentNope + kLatentRope);
constexpr int kValueDim = static_cast<int>(kLatentNope);
constexpr int kTile = 32;   // keys
constexpr int kMostWaves = 8;
constexpr std::size_t kMostStride = std::size_t{1} << 25;  // of a key's row, in numbers
constexpr int kSample = 8;  // keys of a part that give its powers of two
constexpr int kSteps = kKeyDim / 32;    // of the scores' sum
constexpr int kDims = kValueDim / 16;   // tiles of output dims
constexpr int kKeyPitch = kKeyDim * 2;  // bytes of a row of one term in LDS
constexpr int kValuePitch = kValueDim * 2;
// Numbers from here on have an infinite first term.
constexpr float kWild = 0x1.ffp+127f;
// A row's reference stays while no score is above it by more than this (log2
// units): fp16's largest number is 2^16.
constexpr float kSlack = 7.0f;
// fp16 terms: logarithms of the factor on probabilities, and of where the largest
// numbers of queries, keys and values go.
constexpr float kProbLog = 8.0f;
constexpr int kQueryLog = 10;
constexpr int kKeyLog = 4;
constexpr int kValueLog = 8;
// Outputs (of values as scaled) below which 2^-25 may count: it is 2^-21 of them.
constexpr float kSmallOutput = 0x1p-4f;
// What undoes the scores' powers of two must be below this, or this times the row's
// largest score (log2 units): 192 losses of 2^-25 of keys, a third of that each in the
// mean, at queries below 2^11, half that in the mean, are 2^-14 of it in the mean, and
// so 2^-22 of a score.
constexpr float kLargeScores = 0x1p-8f;

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

// A unit to join: one that a group's range ends without starting it.
struct ExpandedJob {
  int b, h, rb;     // sequence (-1: none), head, row block
  int first, last;  // groups whose ranges start and end the unit
};

struct ExpandedStream {
  float* part_o;     // [2 * groups, RB, 128]
  float* part_ml;    // [2 * groups, RB, 2]
  ExpandedJob* jobs; // by unit where there are no more units than groups, else by group
  // A byte a wavefront: 1 if its rows are to be computed again.
  unsigned char* unit_marks;   // [row blocks, batch, heads, waves]: units that a group has whole
  unsigned char* part_marks;   // [2 * groups, waves]: partials
  unsigned char* group_marks;  // [groups, waves]: any of the group's
  int groups;
  int by_unit;
  int weave;  // heads whose units take turns in the list: what a range has units of
};

// Terms of an fp32 number, fp16 or bf16, and the products of two numbers' that are
// taken.
constexpr int terms(bool f16) { return f16 ? 2 : 3; }
constexpr int products(bool f16) { return f16 ? 3 : 6; }

// fp16 terms of x and y, packed into words: the first, of `scale` times the numbers (or
// of the numbers), and the second, what the first one leaves.  A mixed-precision
// instruction a number: the compiler must not see that it adds 0, multiplies by 1, or
// knows a half of the word.
__device__ __forceinline__ unsigned first_half_term(float x, float y, float scale) {
  float zero = 0.0f;
  asm("" : "+s"(zero));
  const v2h h{static_cast<_Float16>(__builtin_fmaf(x, scale, zero)),
              static_cast<_Float16>(__builtin_fmaf(y, scale, zero))};
  unsigned word = __builtin_bit_cast(unsigned, h);
  asm("" : "+v"(word));
  return word;
}
__device__ __forceinline__ unsigned first_half_term(float x, float y) {
  unsigned word = __builtin_bit_cast(unsigned, __builtin_convertvector((v2f{x, y}), v2h));
  asm("" : "+v"(word));
  return word;
}
__device__ __forceinline__ unsigned second_half_term(float x, float y, float scale, unsigned first) {
  const v2h h = __builtin_bit_cast(v2h, first);
  const v2h r{static_cast<_Float16>(__builtin_fmaf(x, scale, -static_cast<float>(h[0]))),
              static_cast<_Float16>(__builtin_fmaf(y, scale, -static_cast<float>(h[1])))};
  return __builtin_bit_cast(unsigned, r);
}
__device__ __forceinline__ unsigned second_half_term(float x, float y, unsigned first) {
  float one = 1.0f;
  asm("" : "+s"(one));
  return second_half_term(x, y, one, first);
}
// The next bf16 term; x and y become what it leaves.
__device__ __forceinline__ unsigned next_bf16_term(float& x, float& y) {
  const unsigned t = __builtin_bit_cast(unsigned, __builtin_convertvector((v2f{x, y}), v2bf));
  x -= __uint_as_float(t << 16);
  y -= __uint_as_float(t & 0xffff0000u);
  return t;
}
// Term `n`; `words` has those before it.
template <bool F16>
__device__ __forceinline__ void next_term(float& x, float& y, int n, unsigned* words) {
  if constexpr (F16) {
    words[n] = n == 0 ? first_half_term(x, y) : second_half_term(x, y, words[0]);
  } else {
    words[n] = next_bf16_term(x, y);
  }
}

// The power of two that puts `most` into [2^to, 2^(to + 1)), as far as it is a normal
// number (1 for 0), and what undoes it.
__device__ __forceinline__ float grow_to(float most, int to, float& unscale) {
  const int e =
      most == 0.f ? to : min(max(static_cast<int>(__float_as_uint(most) >> 23) - 127, -100), 100);
  unscale = __uint_as_float(static_cast<unsigned>(127 - to + e) << 23);
  return __uint_as_float(static_cast<unsigned>(127 + to - e) << 23);
}

// Chunks of 16 bytes are exchanged by row, so that a read of one chunk of 16 rows
// (scores) and of 32 bytes of 8 rows (outputs) hits distinct banks: key rows lie 128
// bytes from a multiple of 256 apart, value rows 256.
__device__ __forceinline__ unsigned key_place(int row, int chunk) {
  const int turn = (row & 2) | ((row & 8) >> 1);
  return static_cast<unsigned>(row * kKeyPitch + (chunk ^ turn) * 16);
}
__device__ __forceinline__ unsigned value_place(int row, int chunk) {
  return static_cast<unsigned>(row * kValuePitch + (chunk ^ (2 * (row & 7))) * 16);
}

// Item i of a range: keys of tile i and values of tile i - 1, what one step takes.  Of
// eight wavefronts four are half a step behind: item i + 2 is on its way while the last
// of item i is read.
template <bool F16>
struct ExpandedShared {
  struct Item {
    __align__(1024) unsigned char k[terms(F16)][kTile * kKeyPitch];
    __align__(1024) unsigned char v[terms(F16)][kTile * kValuePitch];
  };
  static constexpr int kItems = F16 ? 3 : 2;
  Item item[kItems];
  unsigned poison[2][4];  // bf16 terms: keys of the item's values that must not be seen
  // fp16 terms: what undoes the powers of two of an item's keys and values, where a unit's
  // begin with it, by the item's number modulo 4.
  float key_unscale[kMostWaves][4], value_unscale[kMostWaves][4];
};

// What a unit's start costs a workgroup that has begun with another one, in tiles: its
// queries have to come and be split, and the last unit's part is written.  (5 x 20
// heads of up to 257 rows: 42 us with 1, 36 with 2 or 3, 38 with 6.)
constexpr int kStart = 3;

// A place in the flat list, in which each unit has kStart places before its tiles, and
// what of its unit is in the workgroup's range.
struct ExpandedCursor {
  int b, h, rb, blk, to;  // the next tile, and the end of the range's
  int h0;                 // the first head of those woven with it
  int left;               // places of the range behind the unit's
  long long base;         // the unit's first place
  int length, count, nb;
  int first;              // keys that the unit's first row sees
  int bad;                // the length lies outside [0, keys]
};

// Tiles of a unit of sequence b: one at least where it has rows.
template <int RB>
__device__ __forceinline__ int unit_tiles(int length, int count, int rb) {
  const int row0 = rb * RB;
  if (row0 >= count) return 0;
  const int sees = length - count + min(count, row0 + RB);
  return max((sees + kTile - 1) / kTile, 1);
}

// Places of a sequence's row blocks, for each head: the sum over them of unit_tiles and
// kStart.  Of all but the last block the tiles grow by RB / kTile a block, from 1 up.
template <int RB>
__device__ __forceinline__ long long head_places(int length, int count) {
  if (count <= 0) return 0;
  constexpr long long kGrow = RB / kTile;
  const long long blocks = (count + RB - 1) / RB;
  const int before = length - count;
  // (Rounded up, whatever the sign.)
  const long long tiles = before >= 0 ? (before + kTile - 1) / kTile : -(-before / kTile);
  const long long ones = tiles >= 1 ? 0 : min((-tiles) / kGrow, blocks - 1);
  const long long rest = blocks - 1 - ones;
  return ones + rest * tiles + kGrow * (rest * (ones + blocks) / 2) +
         max((length + kTile - 1) / kTile, 1) + kStart * blocks;
}

// A sequence's number of keys (0 where it is none) and of rows.
struct SequenceSize {
  int length, count, bad;
};
__device__ __forceinline__ SequenceSize sequence_size(const ExpandedKernelArgs& a, long long b) {
  SequenceSize s{0, 0, 0};
  if (b >= a.batch) return s;
  s.length = a.key_lengths != nullptr ? a.key_lengths[b] : a.keys;
  s.count = clamped_count(a, static_cast<int>(b));
  s.bad = s.length < 0 || s.length > a.keys;
  if (s.bad != 0) s.length = 0;
  return s;
}

template <int RB>
__device__ __forceinline__ void set_unit(ExpandedCursor& c) {
  c.nb = unit_tiles<RB>(c.length, c.count, c.rb);
  c.first = c.length - c.count + c.rb * RB + 1;
}
template <int RB>
__device__ __forceinline__ void load_unit(const ExpandedKernelArgs& a, ExpandedCursor& c) {
  const int length = a.key_lengths != nullptr ? uniform_read(a.key_lengths + c.b) : a.keys;
  c.bad = length < 0 || length > a.keys;
  c.length = c.bad ? 0 : length;
  c.count = a.tokens;
  if (a.token_counts != nullptr) c.count = min(max(uniform_read(a.token_counts + c.b), 0), a.tokens);
  set_unit<RB>(c);
}

// The range of a workgroup: consecutive ones go to an XCD, which has every eighth
// workgroup.
__device__ __forceinline__ int range_of(int block, int groups) {
  return block % kXcds * (groups / kXcds) + block / kXcds;
}

// Range `group`'s first place, of ranges of `each` places; whether it has a tile.  The
// list goes by sequence, `weave` heads at a time, row block, head of those, and tile:
// ranges of so many units begin a head's row blocks at one time.
template <int RB>
__device__ __forceinline__ bool first_place(const ExpandedKernelArgs& a, const ExpandedStream& st,
                                            int group, int lane, long long& each,
                                            ExpandedCursor& c) {
  const SequenceSize mine = sequence_size(a, lane);
  auto places = [&](const SequenceSize& s) { return head_places<RB>(s.length, s.count) * a.heads; };
  const long long own = places(mine);
  const long long sums = lane_scan(own, lane);
  long long total = uniform_long(__shfl(sums, 63, 64));
  if (a.batch > 64) {
    long long more = 0;
    for (long long b0 = 64; b0 < a.batch; b0 += 64) more += places(sequence_size(a, b0 + lane));
    total += uniform_long(__shfl(lane_scan(more, lane), 63, 64));
  }
  each = uniform_long(max(divide(total + st.groups - 1, st.groups), 1ll));
  const long long g0 = group * each;
  const long long have = min(each, total - g0);
  if (have <= 0) return false;
  long long base = 0;
  for (long long b0 = 0; b0 < a.batch; b0 += 64) {
    const SequenceSize size = b0 == 0 ? mine : sequence_size(a, b0 + lane);
    const long long n = b0 == 0 ? own : places(size);
    const long long sum = b0 == 0 ? sums : lane_scan(n, lane);
    const long long from = base + sum - n, to = base + sum;
    const unsigned long long hit = __ballot(from <= g0 && g0 < to);
    if (hit != 0) {
      const int src = __ffsll(static_cast<long long>(hit)) - 1;
      c.b = __builtin_amdgcn_readfirstlane(static_cast<int>(b0) + src);
      c.length = __builtin_amdgcn_readlane(size.length, src);
      c.count = __builtin_amdgcn_readlane(size.count, src);
      c.bad = __builtin_amdgcn_readlane(size.bad, src);
      base = uniform_long(__shfl(from, src, 64));
      break;
    }
    base += uniform_long(__shfl(sum, 63, 64));
  }
  const long long head = uniform_long(head_places<RB>(c.length, c.count));
  const int woven = __builtin_amdgcn_readfirstlane(
      static_cast<int>(divide(g0 - base, head * st.weave)));
  c.h0 = woven * st.weave;
  base += c.h0 * head;
  const int heads = min(st.weave, a.heads - c.h0);
  for (int rb0 = 0;; rb0 += 64) {
    const int tiles = unit_tiles<RB>(c.length, c.count, rb0 + lane);
    const long long n = tiles > 0 ? static_cast<long long>(tiles + kStart) * heads : 0;
    const long long sum = lane_scan(n, lane);
    const unsigned long long hit = __ballot(base + sum - n <= g0 && g0 < base + sum);
    if (hit != 0 || rb0 >= c.count / RB) {
      const int src = hit != 0 ? __ffsll(static_cast<long long>(hit)) - 1 : 0;
      c.rb = __builtin_amdgcn_readfirstlane(rb0 + src);
      base = uniform_long(base + __shfl(sum - n, src, 64));
      break;
    }
    base += uniform_long(__shfl(sum, 63, 64));
  }
  set_unit<RB>(c);
  const int before = __builtin_amdgcn_readfirstlane(
      static_cast<int>(divide(g0 - base, c.nb + kStart)));
  c.h = c.h0 + before;
  c.base = uniform_long(base + static_cast<long long>(before) * (c.nb + kStart));
  const int in = __builtin_amdgcn_readfirstlane(static_cast<int>(g0 - c.base));
  c.blk = max(in - kStart, 0);
  c.to = __builtin_amdgcn_readfirstlane(
      static_cast<int>(min(static_cast<long long>(c.nb), in + have - kStart)));
  c.left =
      __builtin_amdgcn_readfirstlane(static_cast<int>(max(have - (c.nb + kStart - in), 0ll)));
  return c.to > c.blk;
}

__device__ __forceinline__ std::size_t unit_index(const ExpandedKernelArgs& a,
                                                  const ExpandedCursor& c) {
  return (static_cast<std::size_t>(c.rb) * a.batch + c.b) * a.heads + c.h;
}

// Whether the range has tiles of a later unit, and that unit.
__device__ __forceinline__ bool more_units(const ExpandedCursor& c) { return c.left > kStart; }
template <int RB>
__device__ __forceinline__ void next_unit(const ExpandedKernelArgs& a, const ExpandedStream& st,
                                          ExpandedCursor& c) {
  c.base += c.nb + kStart;
  if (++c.h == min(c.h0 + st.weave, a.heads)) {
    c.h = c.h0;
    if (++c.rb * RB >= c.count) {
      c.rb = 0;
      c.h = c.h0 = c.h0 + st.weave;
      if (c.h0 >= a.heads) {
        c.h = c.h0 = 0;
        do {
          ++c.b;
          load_unit<RB>(a, c);
        } while (c.nb == 0);
      }
    }
  }
  set_unit<RB>(c);
  c.blk = 0;
  c.to = min(c.nb, c.left - kStart);
  c.left = max(c.left - c.nb - kStart, 0);
}

// The range that begins at `cur`.  RT tiles of 16 query rows a wavefront, units of RB
// rows.  F16: which terms (bf16 ones compute again, and mark nothing).  `each`:
// places of a range.
template <int WAVES, int RT, bool F16>
__device__ __forceinline__ void expanded_range(const ExpandedKernelArgs& a, const ExpandedStream& st,
                                               ExpandedShared<F16>& sh, ExpandedCursor cur,
                                               long long each) {
  constexpr int RB = 16 * WAVES * RT;
  constexpr int kTerms = terms(F16), kProducts = products(F16);
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, grp = lane >> 4;
  const int group = range_of(static_cast<int>(blockIdx.x), st.groups);
  auto barrier = [] {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };

  // ---- staging: of a key and of a value, a thread has chunks of eight numbers, kLanes
  // apart, and of the shared part one of kShared numbers.
  constexpr int kLanes = 64 * WAVES / kTile;
  constexpr int kOwn = kValueDim / 8 / kLanes, kShared = static_cast<int>(kLatentRope) / kLanes;
  constexpr int kPieces = 2 * kOwn + 1;
  const int srow = tid / kLanes, part = tid % kLanes;
  struct Source {  // a tile: its first rows
    const float* k;
    const float* r;
    const float* v;
    int last;   // its last key, or a later one, in the sequence: -1 if that is empty
    int seen;   // its keys that every row of the unit sees: a later one's number too, or < 0
    int opens;  // the first tile of its unit in the range
  };
  auto source = [&](const ExpandedCursor& c) {
    Source s{};
    const std::size_t j = static_cast<std::size_t>(c.blk) * kTile;
    // (Of an empty sequence nothing is there, and nothing of it is used: a query's
    // numbers are.)
    s.k = s.r = s.v = a.query + static_cast<std::size_t>(c.b) * a.query_at.batch;
    if (c.length > 0) {
      s.k = a.key + static_cast<std::size_t>(c.b) * a.key_at.batch +
            static_cast<std::size_t>(c.h) * a.key_at.head + j * a.key_at.token;
      s.r = a.rope_key + static_cast<std::size_t>(c.b) * a.rope_at.batch + j * a.rope_at.token;
      s.v = a.value + static_cast<std::size_t>(c.b) * a.value_at.batch +
            static_cast<std::size_t>(c.h) * a.value_at.head + j * a.value_at.token;
    }
    s.last = c.length - 1 - c.blk * kTile;
    s.seen = c.first - c.blk * kTile;
    s.opens = 1;
    return s;
  };
  // What the registers hold, or are sent for: keys of a tile, and values of the one
  // before.
  Source keys = source(cur), values = keys;
  values.opens = 0;
  v4f raw_k[kOwn + 1][2], raw_v[kOwn][2];  // (a key's last chunk is the shared part's)
  // Bytes from a tile's first row, 32 bits: a row's stride is below kMostStride.
  auto row_offset = [&](int last, std::size_t stride, int numbers) {
    const unsigned row = static_cast<unsigned>(max(min(srow, last), 0));
    return (__umul24(row, static_cast<unsigned>(stride / 4)) + static_cast<unsigned>(part * numbers / 4)) *
           16u;
  };
  // Chunk i: a key's, then a value's.
  auto fetch = [&](int i) {
    const float* const base = i < kOwn ? keys.k : i == kOwn ? keys.r : values.v;
    const unsigned offset = i < kOwn    ? row_offset(keys.last, a.key_at.token, 8)
                            : i == kOwn ? row_offset(keys.last, a.rope_at.token, kShared)
                                        : row_offset(values.last, a.value_at.token, 8);
    const auto* const from = reinterpret_cast<const unsigned char*>(base) + offset +
                             (i < kOwn ? i : i == kOwn ? 0 : i - kOwn - 1) * kLanes * 32;
#pragma unroll
    for (int w = 0; w < (i == kOwn ? kShared / 4 : 2); ++w) {
      const v4f x = *reinterpret_cast<const v4f*>(from + 16 * w);
      if (i <= kOwn) {
        raw_k[i <= kOwn ? i : 0][w] = x;
      } else {
        raw_v[i <= kOwn ? 0 : i - kOwn - 1][w] = x;
      }
    }
  };
  // fp16 terms: the powers of two of the keys and values on their way, and the next
  // unit's of the values.
  float key_scale = 1.f, value_scale = 1.f, next_value_scale = 1.f, next_value_unscale = 1.f;
  // Those of the unit that begins with the keys on their way, by the first of its keys
  // that all its rows see.  Each wavefront finds them for itself.
  auto sample = [&](int item) {
    const Source& s = keys;
    const int have = min(min(s.seen, s.last + 1), kSample);
    float top[2] = {0.f, 0.f};
    if (have > 0) {
      const int r = lane / kSample, c = lane % kSample;
      const std::size_t j = static_cast<std::size_t>(min(r, have - 1));
      const float* const k = s.k + j * a.key_at.token + 4 * c;
      const float* const rope = s.r + j * a.rope_at.token + 4 * c;
      const float* const v = s.v + j * a.value_at.token + 4 * c;
      auto take = [](float& most, v4f x) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float y = fabsf(x[e]);
          most = fmaxf(most, y < 0x1p100f ? y : 0.f);
        }
      };
#pragma unroll
      for (int i = 0; i < kValueDim; i += 4 * kSample) {
        take(top[0], *reinterpret_cast<const v4f*>(k + i));
        take(top[1], *reinterpret_cast<const v4f*>(v + i));
      }
#pragma unroll
      for (int i = 0; i < static_cast<int>(kLatentRope); i += 4 * kSample) {
        take(top[0], *reinterpret_cast<const v4f*>(rope + i));
      }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int bit = 32; bit >= 1; bit /= 2) top[i] = fmaxf(top[i], __shfl_xor(top[i], bit, 64));
    }
    float key_un;
    key_scale = grow_to(top[0], kKeyLog, key_un);
    next_value_scale = grow_to(top[1], kValueLog, next_value_unscale);
    if (lane == 0) sh.key_unscale[wave][item & 3] = key_un;
  };
  // The way into LDS in small parts, each one term of two numbers: a chunk's pairs of
  // numbers, then the next chunk's; its last part writes it.
  constexpr int kPairs = 2 * kOwn * 4 + kShared / 2;
  constexpr int kStageParts = kPairs * kTerms;
  unsigned words[4][kTerms];
  float sx = 0.f, sy = 0.f;
  auto stage = [&](int buf, int i) {
    const int level = i % kTerms, at = i / kTerms;
    const bool before = at < 4 * kOwn, shared = !before && at < 4 * kOwn + kShared / 2;
    const int in = before || shared ? at : at - kShared / 2 + 4;  // (as if all had four pairs)
    const int chunk = in / 4, pair = in % 4;
    if (level == 0) {
      const v4f x = chunk <= kOwn ? raw_k[chunk <= kOwn ? chunk : 0][pair / 2]
                                  : raw_v[chunk <= kOwn ? 0 : chunk - kOwn - 1][pair / 2];
      sx = x[2 * (pair % 2)];
      sy = x[2 * (pair % 2) + 1];
    }
    if constexpr (F16) {
      const float by = chunk <= kOwn ? key_scale : value_scale;
      words[pair][level] = level == 0 ? first_half_term(sx, sy, by)
                                      : second_half_term(sx, sy, by, words[pair][0]);
    } else {
      words[pair][level] = next_bf16_term(sx, sy);
    }
    if (pair != (shared ? kShared / 2 : 4) - 1 || level != kTerms - 1) return;
    fetch(chunk);
    auto& into = sh.item[buf];
    unsigned char* const to =
        chunk < kOwn    ? into.k[0] + key_place(srow, part + kLanes * chunk)
        : chunk == kOwn ? into.k[0] + key_place(srow, 16 + part * kShared / 8) +
                              part * kShared * 2 % 16
                        : into.v[0] + value_place(srow, part + kLanes * (chunk - kOwn - 1));
    const unsigned plane = chunk <= kOwn ? kTile * kKeyPitch : kTile * kValuePitch;
#pragma unroll
    for (int n = 0; n < kTerms; ++n) {
      if (shared && kShared == 4) {
        *reinterpret_cast<v2u*>(to + n * plane) = v2u{words[0][n], words[1][n]};
      } else {
        *reinterpret_cast<v4u*>(to + n * plane) =
            v4u{words[0][n], words[1][n], words[2][n], words[3][n]};
      }
    }
  };
  // bf16 terms: values of keys that some row of the unit does not see must be finite: those
  // behind the sequence's last become 0, and of the others those with terms that are
  // not; the latter's keys are noted.
  auto clean_values = [&](int buf, const Source& s) {
    static_assert(F16 || kLanes == 8, "eight threads a key");
    unsigned poison = 0;
    if (kTile > s.seen) {
      bool wild = false;
#pragma unroll
      for (int i = 0; i < kOwn; ++i)
#pragma unroll
        for (int w = 0; w < 2; ++w)
#pragma unroll
          for (int n = 0; n < 4; ++n) wild = wild || !(fabsf(raw_v[i][w][n]) < kWild);
      const unsigned long long hit = __ballot(wild && srow >= s.seen && srow <= s.last);
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        if (((hit >> (8 * r)) & 0xffull) != 0) poison |= 1u << (8 * wave + r);
      }
      const bool wipe = srow > s.last || ((poison >> (srow & 31)) & 1u) != 0;
#pragma unroll
      for (int i = 0; i < kOwn; ++i)
#pragma unroll
        for (int w = 0; w < 2; ++w)
#pragma unroll
          for (int n = 0; n < 4; ++n) raw_v[i][w][n] = wipe ? 0.f : raw_v[i][w][n];
    }
    if (lane == 0) sh.poison[buf][wave] = poison;
  };

  // ---- the wavefront's rows of a unit: tile t's row `col`.
  auto unit_row = [&](int t) { return (wave * RT + t) * 16 + col; };
  v4u q[kSteps][RT][kTerms];
  v4f o[RT][kDims];  // o[t][dt][i]: dim 16 dt + 4 grp + i of row col
  float m[RT], l[RT];
  float unscale[RT];  // fp16 terms: what undoes the row's power of two and the keys'
  int limit[RT];      // keys that the row sees
  auto start = [&](const ExpandedCursor& c, float key_un) {
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      const int row = c.rb * RB + unit_row(t);
      const bool live = row < c.count;
      limit[t] = c.length - c.count + row + 1;
      const float* const src = a.query + static_cast<std::size_t>(c.b) * a.query_at.batch +
                               static_cast<std::size_t>(c.h) * a.query_at.head +
                               static_cast<std::size_t>(live ? row : 0) * a.query_at.token;
      v4f x[kSteps][2];
#pragma unroll
      for (int s = 0; s < kSteps; ++s)
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          x[s][w] = *reinterpret_cast<const v4f*>(src + 32 * s + 8 * grp + 4 * w);
        }
      float grow = a.qscale;
      unscale[t] = 1.f;
      if constexpr (F16) {
        float top = 0.f;
#pragma unroll
        for (int s = 0; s < kSteps; ++s)
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            const v4f y = x[s][w];
            top = fmaxf(top, fmaxf(fmaxf(fabsf(y[0]), fabsf(y[1])), fmaxf(fabsf(y[2]), fabsf(y[3]))));
          }
        grow = grow_to(row_max(top), kQueryLog, unscale[t]);
        // (Positive, or scores of -infinity would not stay that: the score scale's
        // sign goes with the queries, which a scale of 0 makes 0.)
        grow = a.qscale > 0.f ? grow : a.qscale < 0.f ? -grow : 0.f;
        unscale[t] = fmaxf(unscale[t] * fabsf(a.qscale) * key_un, 1.2e-38f);
      }
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        unsigned w[4][kTerms];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float y0 = x[s][i >> 1][2 * (i & 1)] * grow, y1 = x[s][i >> 1][2 * (i & 1) + 1] * grow;
#pragma unroll
          for (int n = 0; n < kTerms; ++n) next_term<F16>(y0, y1, n, w[i]);
        }
#pragma unroll
        for (int i = 0; i < kTerms; ++i) {
          q[s][t][i] = v4u{w[0][i], w[1][i], w[2][i], w[3][i]};
          // (Queries live in the accumulation registers, all else in the others.)
          asm("" : "+a"(q[s][t][i]));
        }
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int dt = 0; dt < kDims; ++dt) o[t][dt] = v4f{0.f, 0.f, 0.f, 0.f};
      m[t] = live ? -INFINITY : INFINITY;  // (a row that is none never moves the others)
      l[t] = 0.f;
    }
  };

  // A matrix instruction takes 16 cycles, of which its issue takes 4: the RT ones of a
  // product have other work put behind them, a part at a time.  (In one piece before
  // or behind the products of a step, which is how the compiler would have it, the two
  // add up: two matrix and four other instructions take 41 cycles in turn, eight others
  // in one piece 50 by themselves.)
  auto product = [](int sum, int i) {  // its place in the order below
    return kProducts - (sum + 1) * (sum + 2) / 2 + sum - i;
  };

  // Scores of a tile: sc[t][h][i] is key 16 h + 4 grp + i of tile t's row col.
  unsigned key_at[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) key_at[i] = key_place(col, 4 * i + grp);
  auto scores = [&](int buf, v4f (&sc)[RT][2], auto&& beside) {
    v4u k[2][kTerms];
    auto read = [&](int u) {  // dims 32 (u / 2) and on of keys 16 (u % 2) and on
      const int s = u / 2, h = u % 2;
#pragma unroll
      for (int i = 0; i < kTerms; ++i) {
        // (Rows 16 and on are exchanged as rows 0 and on.)
        k[u % 2][i] = *reinterpret_cast<const v4u*>(sh.item[buf].k[i] + key_at[s % 2] +
                                                    (s / 2) * 128 + h * (16 * kKeyPitch));
      }
    };
    read(0);
    read(1);
#pragma unroll
    for (int t = 0; t < RT; ++t) sc[t][0] = sc[t][1] = v4f{0.f, 0.f, 0.f, 0.f};
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int u = 0; u < 2 * kSteps; ++u) {
      const int s = u / 2, h = u % 2;
      // Smallest products first.
#pragma unroll
      for (int sum = kTerms - 1; sum >= 0; --sum)
#pragma unroll
        for (int i = sum; i >= 0; --i) {
#pragma unroll
          for (int t = 0; t < RT; ++t) sc[t][h] = matrix_step<F16>(k[u % 2][i], q[s][t][sum - i], sc[t][h]);
          beside(kProducts * u + product(sum, i));
          __builtin_amdgcn_sched_barrier(0);
        }
      if (u + 2 < 2 * kSteps) read(u + 2);
    }
  };
  // A row's reference follows the tile's largest score where that is far above it.  (By
  // the row's own scores alone: no bit of it depends on keys that only others see.)
  auto follow = [&](const v4f (&sc)[RT][2]) {
    float mx[RT];
    bool above = false;
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      const v4f x = sc[t][0], y = sc[t][1];
      mx[t] = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])),
                    fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3])));
      if constexpr (F16) mx[t] *= unscale[t];
      above = above || mx[t] > m[t] + kSlack;
    }
    if (__ballot(above) != 0) {
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        const float most = row_max(mx[t]);
        const float mn = most > m[t] + kSlack ? most : m[t];
        const float alpha = exp2_ratio(m[t], mn);
#pragma unroll
        for (int dt = 0; dt < kDims; ++dt) o[t][dt] *= alpha;
        l[t] *= alpha;
        m[t] = mn;
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  };
  // Scores of keys that a row does not see become -infinity, and NaN where `poison`
  // has one that it sees.
  auto mask = [&](int first, unsigned poison, v4f (&sc)[RT][2]) {
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int n = 16 * h + 4 * grp + i;
          float x = sc[t][h][i];
          if (((poison >> n) & 1u) != 0) x = NAN;
          sc[t][h][i] = first + n < limit[t] ? x : -INFINITY;
        }
  };
  struct Probabilities {
    unsigned w[RT][4][kTerms];
  };
  // In small parts: of two keys their exponentials, then a term each.
  constexpr int kProbParts = RT * 4 * (1 + kTerms);
  float py0 = 0.f, py1 = 0.f;
  auto probability = [&](int i, const v4f (&sc)[RT][2], const float (&ref)[RT], Probabilities& p) {
    const int pair = i / (1 + kTerms), level = i % (1 + kTerms), t = pair / 4, n = pair % 4;
    if (level == 0) {
      const float x = sc[t][n / 2][2 * (n % 2)], y = sc[t][n / 2][2 * (n % 2) + 1];
      if constexpr (F16) {
        py0 = __builtin_amdgcn_exp2f(__builtin_fmaf(x, unscale[t], -ref[t]));
        py1 = __builtin_amdgcn_exp2f(__builtin_fmaf(y, unscale[t], -ref[t]));
      } else {
        py0 = __builtin_amdgcn_exp2f(x - ref[t]);
        py1 = __builtin_amdgcn_exp2f(y - ref[t]);
      }
      return;
    }
    if (level == 1) l[t] += py0 + py1;
    next_term<F16>(py0, py1, level - 1, p.w[t][n]);
  };
  const int vrow = 4 * grp + (col >> 2);
  unsigned value_at[4];
#pragma unroll
  for (int d = 0; d < 4; ++d) {
    value_at[d] = value_place(vrow, 2 * d + ((col >> 1) & 1)) + (col & 1) * 8u;
  }
  auto add_values = [&](int buf, const Probabilities& p, auto&& beside) {
    using LdsV4s = __attribute__((address_space(3))) v4s;
    v4u pop[RT][kTerms];
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
      for (int i = 0; i < kTerms; ++i) {
        pop[t][i] = v4u{p.w[t][0][i], p.w[t][1][i], p.w[t][2][i], p.w[t][3][i]};
      }
    v4u v[2][kTerms];
    auto read = [&](int dt) {
#pragma unroll
      for (int i = 0; i < kTerms; ++i) {
        // (Chunks 8 and on lie where chunks 0 and on do, exchanged in their group.)
        const unsigned char* const from = sh.item[buf].v[i] + (value_at[dt % 4] ^ (dt / 4 * 128u));
        const v4s v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsV4s*)(from));
        const v4s v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsV4s*)(from + 16 * kValuePitch));
        v[dt % 2][i] = __builtin_bit_cast(v4u, __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7));
      }
    };
    read(0);
    read(1);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int dt = 0; dt < kDims; ++dt) {
#pragma unroll
      for (int sum = kTerms - 1; sum >= 0; --sum)
#pragma unroll
        for (int i = sum; i >= 0; --i) {
#pragma unroll
          for (int t = 0; t < RT; ++t) o[t][dt] = matrix_step<F16>(v[dt % 2][i], pop[t][sum - i], o[t][dt]);
          beside(kProducts * dt + product(sum, i));
          __builtin_amdgcn_sched_barrier(0);
        }
      if (dt + 2 < kDims) read(dt + 2);
    }
  };

  // ---- the range.  Step n: scores of tile n + 1 beside tile n's probabilities, tile
  // n's outputs beside the way of item n + 2 into LDS; behind each chunk's way, that of
  // item n + 3 is sent for.
  ExpandedCursor ahead = cur;  // the tile whose keys are sent for
  // Keys of the next tile and values of the one before.  (Behind the range the last
  // one again, which no one reads.)
  auto advance = [&] {
    values = keys;
    keys.opens = 0;
    if (ahead.blk + 1 < ahead.to) {
      ++ahead.blk;
      keys.k += kTile * a.key_at.token;
      keys.r += kTile * a.rope_at.token;
      keys.v += kTile * a.value_at.token;
      keys.last -= kTile;
      keys.seen -= kTile;
    } else if (more_units(ahead)) {
      next_unit<RB>(a, st, ahead);
      keys = source(ahead);
    }
  };
  // Before item i's way into LDS, into `buf`: its powers of two, or its values made
  // finite.
  auto ready = [&](int i, int buf) {
    if constexpr (F16) {
      if (values.opens != 0) {
        value_scale = next_value_scale;
        if (lane == 0) sh.value_unscale[wave][i & 3] = next_value_unscale;
      }
      if (keys.opens != 0) sample(i);
    } else {
      clean_values(buf, values);
    }
  };
  // Items 0 and 1.  (Item 0's values, the first tile's, are not read.)
#pragma unroll
  for (int item = 0; item < 2; ++item) {
    if (item == 0) {
#pragma unroll
      for (int i = 0; i < kPieces; ++i) fetch(i);
    }
    ready(item, item);
    advance();
#pragma unroll
    for (int i = 0; i < kStageParts; ++i) stage(item, i);
  }
  barrier();
  constexpr int kItems = ExpandedShared<F16>::kItems;
  constexpr bool kBehind = WAVES == 8;  // whether four wavefronts are half a step behind
  int n = 0, slot = 0;  // n modulo kItems
  auto later = [](int at, int by) { return at + by >= kItems ? at + by - kItems : at + by; };
  for (;;) {
    start(cur, F16 ? sh.key_unscale[wave][n & 3] : 1.f);
    const float value_un = F16 ? sh.value_unscale[wave][(n + 1) & 3] : 1.f;
    const int from = cur.blk, to = cur.to;
    const int whole = max(cur.first, 0) / kTile;  // tiles before are seen by every row
    v4f sc[RT][2];
    scores(slot, sc, [](int) {});
    // (Of two items, this one's keys are taken before it is written again.)
    if constexpr (kItems == 2) barrier();
    if (kBehind && n == 0 && wave >= 4) barrier();
    for (int blk = from; blk < to; ++blk) {
      const int buf = later(slot, 1), into = later(slot, 2);
      if (blk >= whole) {
        unsigned poison = 0;
        if constexpr (!F16) {
          poison = sh.poison[buf][0] | sh.poison[buf][1] | sh.poison[buf][2] | sh.poison[buf][3];
        }
        mask(blk * kTile, poison, sc);
      }
      follow(sc);
      float ref[RT];
#pragma unroll
      for (int t = 0; t < RT; ++t) ref[t] = (m[t] == -INFINITY ? 0.f : m[t]) - (F16 ? kProbLog : 0.f);
      ready(n + 2, into);
      advance();
      Probabilities p;
      // Of the way into LDS, the parts beside the scores: those that their steps have room
      // for, or, where wavefronts are half a step behind, the keys', which the others
      // read first.
      constexpr int kKeyParts = (4 * kOwn + kShared / 2) * kTerms;
      constexpr int kRoom = 2 * kSteps * kProducts - kProbParts;
      constexpr int kBeside = kBehind ? kKeyParts : kRoom < kStageParts ? kRoom : kStageParts;
      static_assert(kBeside <= kRoom, "a slot a part");
      if (blk + 1 < to) {
        v4f last[RT][2];
#pragma unroll
        for (int t = 0; t < RT; ++t)
#pragma unroll
          for (int h = 0; h < 2; ++h) last[t][h] = sc[t][h];
        // (A copy that the compiler does not know, or it takes the exponentials of both
        // cases out in front.)
        float ref_here[RT];
#pragma unroll
        for (int t = 0; t < RT; ++t) {
          ref_here[t] = ref[t];
          asm("" : "+v"(ref_here[t]));
        }
        scores(buf, sc, [&](int i) {
          if (i < kBeside) {
            stage(into, i);
          } else if (i - kBeside < kProbParts) {
            probability(i - kBeside, last, ref_here, p);
          }
          if (kBehind && i == kBeside - 1) barrier();
        });
      } else {
#pragma unroll
        for (int i = 0; i < kBeside; ++i) stage(into, i);
        if (kBehind) barrier();
#pragma unroll
        for (int i = 0; i < kProbParts; ++i) probability(i, sc, ref, p);
      }
      add_values(buf, p, [&](int i) {
        constexpr int kLeft = kStageParts - kBeside, kSlots = kDims * kProducts;
#pragma unroll
        for (int j = i * kLeft / kSlots; j < (i + 1) * kLeft / kSlots; ++j) stage(into, kBeside + j);
      });
      ++n;
      slot = buf;
      barrier();
    }
    // The part's end.
    const bool starts = from == 0, ends = to == cur.nb, complete = starts && ends;
    const int partial = 2 * group + (starts ? 1 : 0);
    // (A number that does not fit has terms of infinity and of less that: their sum is NaN.)
    bool wrong = false;
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      const float sum = row_sum(l[t]);
      const int local = unit_row(t), row = cur.rb * RB + local;
      if (F16) {
        float top = 0.f;
        bool nan = !(sum < INFINITY);
#pragma unroll
        for (int dt = 0; dt < kDims; ++dt)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            top = fmaxf(top, fabsf(o[t][dt][i]));
            nan = nan || !(fabsf(o[t][dt][i]) < INFINITY);
          }
        top = row_max(top);
        // (An empty row beside a NaN is computed again too: 0 times it is not 0.)
        const bool lost = sum != 0.f && (top < kSmallOutput * sum ||
                                         unscale[t] > kLargeScores * fmaxf(fabsf(m[t]), 1.f));
        wrong = wrong || (row < cur.count && (nan || lost));
      }
      if (row >= cur.count) continue;
      const bool some = from * kTile < limit[t];  // of the part's keys
      float f = F16 ? value_un : 1.0f;
      if (complete) f = cur.bad != 0 ? NAN : row_factor(sum, some, f);
      float* const dst =
          (complete ? a.out + static_cast<std::size_t>(cur.b) * a.out_at.batch +
                          static_cast<std::size_t>(cur.h) * a.out_at.head +
                          static_cast<std::size_t>(row) * a.out_at.token
                    : st.part_o + (static_cast<std::size_t>(partial) * RB + local) * kValueDim) +
          4 * grp;
#pragma unroll
      for (int dt = 0; dt < kDims; ++dt) *reinterpret_cast<v4f*>(dst + 16 * dt) = o[t][dt] * f;
      if (!complete && grp == 0) {
        float* const ml = st.part_ml + (static_cast<std::size_t>(partial) * RB + local) * 2;
        ml[0] = sum == 0.f && some ? kNoWeights : m[t];
        ml[1] = cur.bad != 0 ? NAN : sum;
      }
    }
    if constexpr (F16) {
      const bool any = __ballot(wrong) != 0;
      if (lane == 0) {
        unsigned char* const mark =
            complete ? st.unit_marks + unit_index(a, cur) * WAVES : st.part_marks + partial * WAVES;
        mark[wave] = any ? 1 : 0;
        if (any) st.group_marks[group * WAVES + wave] = 1;
      }
      if (tid == 0) {
        if (ends && (!starts || st.by_unit != 0)) {
          st.jobs[st.by_unit != 0 ? unit_index(a, cur) : static_cast<std::size_t>(group)] =
              ExpandedJob{starts ? -1 : cur.b, cur.h, cur.rb,
                          static_cast<int>(divide(cur.base + kStart, each)), group};
        }
      }
    }
    if (!more_units(cur)) break;
    next_unit<RB>(a, st, cur);
  }
  if (kBehind && wave < 4) barrier();
  if constexpr (!F16) barrier();  // (another unit may follow)
}

template <int WAVES>
__global__ __launch_bounds__(64 * WAVES) __attribute__((amdgpu_waves_per_eu(WAVES / 4, WAVES / 4)))
    void expanded_kernel(ExpandedKernelArgs a, ExpandedStream st) {
  __shared__ ExpandedShared<true> sh;
  constexpr int RB = 16 * WAVES;
  const int group = range_of(static_cast<int>(blockIdx.x), st.groups);
  if (threadIdx.x == 0 && st.by_unit == 0) st.jobs[group] = ExpandedJob{-1, 0, 0, 0, 0};
  if (threadIdx.x % 64 == 0) st.group_marks[group * WAVES + threadIdx.x / 64] = 0;
  ExpandedCursor cur{};
  long long each;
  if (!first_place<RB>(a, st, group, static_cast<int>(threadIdx.x) & 63, each, cur)) return;
  expanded_range<WAVES, 1, true>(a, st, sh, cur, each);
}

// The same ranges' parts of units that are marked, again.
template <int RT>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(1, 1)))
    void expanded_redo_kernel(ExpandedKernelArgs a, ExpandedStream st) {
  __shared__ ExpandedShared<false> sh;
  constexpr int RB = 64 * RT;
  const int tid = static_cast<int>(threadIdx.x);
  // (Marks of the wavefronts that had a unit, in one word.)
  using Marks = std::conditional_t<RT == 2, unsigned long long, unsigned>;
  const auto* const unit_marks = reinterpret_cast<const Marks*>(st.unit_marks);
  const auto* const part_marks = reinterpret_cast<const Marks*>(st.part_marks);
  const auto* const group_marks = reinterpret_cast<const Marks*>(st.group_marks);
  static_assert(sizeof(Marks) == 4 * RT, "a byte a wavefront");
  bool marked = false;
  for (int g = tid; g < st.groups; g += 256) marked = marked || group_marks[g] != 0;
  if (__syncthreads_or(marked) == 0) return;
  ExpandedCursor cur{};
  long long each;
  if (!first_place<RB>(a, st, range_of(static_cast<int>(blockIdx.x), st.groups), tid & 63, each, cur)) return;
  for (;;) {
    // A unit in several parts is marked if one of them is.
    bool mark = false;
    if (cur.blk == 0 && cur.to == cur.nb) {
      mark = unit_marks[unit_index(a, cur)] != 0;
    } else {
      const int first = static_cast<int>((cur.base + kStart) / each);
      const int last = static_cast<int>((cur.base + kStart + cur.nb - 1) / each);
      for (int g = first + tid; g <= last; g += 256) {
        mark = mark || part_marks[2 * g + (g == first ? 1 : 0)] != 0;
      }
    }
    if (__syncthreads_or(mark) != 0) {
      ExpandedCursor one = cur;
      one.left = 0;
      expanded_range<4, RT, false>(a, st, sh, one, each);
    }
    if (!more_units(cur)) break;
    next_unit<RB>(a, st, cur);
  }
}

// Joins the partials of the units that cross ranges: the first group's second slot
// and the later groups' first ones.  blockIdx.x is a unit or a group; 16 lanes take a
// row, 8 dims each.  A workgroup has `wg_rows` rows, 16 or 4.
constexpr int kFewParts = 16;
__global__ __launch_bounds__(256) void expanded_merge_kernel(ExpandedKernelArgs a, ExpandedStream st,
                                                             int rb_rows, int wg_rows) {
  __shared__ v4f sums[4][64][2];
  __shared__ float totals[4][4];
  const int lane = threadIdx.x & 63, part = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  if (st.by_unit != 0) {  // (of units without rows no one says anything)
    const int entry = static_cast<int>(blockIdx.x) / a.heads;
    if (entry / a.batch * rb_rows >= clamped_count(a, entry % a.batch)) return;
  }
  const ExpandedJob job = st.jobs[blockIdx.x];
  if (job.b < 0) return;
  const int parts = job.last - job.first + 1;
  const int count = clamped_count(a, job.b);
  const int local0 = static_cast<int>(blockIdx.y) * wg_rows;
  auto slot_of = [&](int i, int row) {
    return static_cast<std::size_t>(2 * (job.first + i) + (i == 0 ? 1 : 0)) * rb_rows + row;
  };
  auto finish = [&](int row, const v4f (&o)[2], float sum) {
    const float f = row_factor(sum, false, 1.0f);
    auto* const dst = reinterpret_cast<v4f*>(
                          a.out + static_cast<std::size_t>(job.b) * a.out_at.batch +
                          static_cast<std::size_t>(job.h) * a.out_at.head +
                          static_cast<std::size_t>(job.rb * rb_rows + row) * a.out_at.token) +
                      2 * part;
    dst[0] = o[0] * f;
    dst[1] = o[1] * f;
  };
  if (parts > kFewParts) {
    // Many parts: the wavefronts have every fourth one of the same four rows.
    for (int q = 0; q < wg_rows; q += 4) {
      const int local = local0 + q + (lane >> 4);
      const bool live = local < rb_rows && job.rb * rb_rows + local < count;
      const int row = live ? local : 0;
      float top = -INFINITY;
      for (int i = part; i < parts; i += 16) top = fmaxf(top, st.part_ml[2 * slot_of(i, row)]);
#pragma unroll
      for (int k = 8; k > 0; k /= 2) top = fmaxf(top, __shfl_xor(top, k, 64));
      float sum = 0.f;
      v4f o[2] = {v4f{0.f, 0.f, 0.f, 0.f}, v4f{0.f, 0.f, 0.f, 0.f}};
      constexpr int U = 4;
      for (int i0 = wave; i0 < parts; i0 += 4 * U) {
        v4f x[U][2];
        v2f ml[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const std::size_t at = slot_of(min(i0 + 4 * u, parts - 1), row);
          ml[u] = *reinterpret_cast<const v2f*>(st.part_ml + 2 * at);
          const auto* from = reinterpret_cast<const v4f*>(st.part_o + at * kValueDim) + 2 * part;
          x[u][0] = from[0];
          x[u][1] = from[1];
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          // (A part that saw nothing has no outputs to speak of.)
          if (i0 + 4 * u >= parts) continue;
          const float w = ml[u][1] != 0.f ? exp2_ratio(ml[u][0], top) : 0.f;
          if (w != 0.f) {
            o[0] += x[u][0] * w;
            o[1] += x[u][1] * w;
          }
          sum += part_sum(ml[u][0], ml[u][1], w, top);
        }
      }
      __syncthreads();
      sums[wave][lane][0] = o[0];
      sums[wave][lane][1] = o[1];
      if (part == 0) totals[wave][lane >> 4] = sum;
      __syncthreads();
      if (wave == 0 && live) {
#pragma unroll
        for (int w = 1; w < 4; ++w) {
          o[0] += sums[w][lane][0];
          o[1] += sums[w][lane][1];
          sum += totals[w][lane >> 4];
        }
        finish(local, o, sum);
      }
    }
    return;
  }
  if (wave * 4 >= wg_rows) return;
  const int local = local0 + wave * 4 + (lane >> 4);
  const bool live = local < rb_rows && job.rb * rb_rows + local < count;
  if (__ballot(live) == 0) return;
  const int at = live ? local : 0;
  auto slot = [&](int i) { return slot_of(i, at); };
  // Four partials at a time on their way, the first ones before their weights are known.
  v4f x[4][2];
  auto load = [&](int i0) {
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const auto* from = reinterpret_cast<const v4f*>(
                             st.part_o + slot(min(i0 + u, parts - 1)) * kValueDim) +
                         2 * part;
      x[u][0] = from[0];
      x[u][1] = from[1];
    }
  };
  load(0);
  // A lane of the row has a partial's maximum and sum.
  static_assert(kFewParts <= 16, "16 lanes a row");
  float pm = -INFINITY, pl = 0.f;
  if (live && part < parts) {
    const v2f ml = *reinterpret_cast<const v2f*>(st.part_ml + 2 * slot(part));
    pm = ml[0];
    pl = ml[1];
  }
  float top = pm;
#pragma unroll
  for (int k = 8; k > 0; k /= 2) top = fmaxf(top, __shfl_xor(top, k, 64));
  // (A part that saw nothing has no outputs to speak of.)
  const float w = pl == 0.f ? 0.f : exp2_ratio(pm, top);
  float sum = part_sum(pm, pl, w, top);
#pragma unroll
  for (int k = 8; k > 0; k /= 2) sum += __shfl_xor(sum, k, 64);
  v4f o[2] = {v4f{0.f, 0.f, 0.f, 0.f}, v4f{0.f, 0.f, 0.f, 0.f}};
  for (int i = 0; i < parts; i += 4) {
    if (i != 0) load(i);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const float wi = __shfl(w, (lane & 48) + min(i + u, parts - 1), 64);
      if (i + u < parts && wi != 0.f) {
        o[0] += x[u][0] * wi;
        o[1] += x[u][1] * wi;
      }
    }
  }
  if (live) finish(local, o, sum);
}

// ----------------------------------------------------------------- host ----
constexpr std::size_t kGroups = 256;  // a workgroup a CU: a wavefront a SIMD, for its registers

// Units of 64 rows (four wavefronts) where there are no more: 16 x 16 heads, 64 rows
// over 2048 keys take 134 us, in units of 128 152; 4 x 32 heads, 512 rows over 4096 keys
// take 545 in units of 128, 850 in units of 64, whose keys are split twice as often.
struct ExpandedLayout {
  ExpandedLayout(std::size_t batch, std::size_t heads, std::size_t tokens) {
    rb = tokens <= 64 ? 64 : 128;
    row_blocks = (tokens + rb - 1) / rb;
    auto take = [&](std::size_t n) {
      const std::size_t at = bytes;
      bytes += align256(n);
      return at;
    };
    jobs = take(kGroups * sizeof(ExpandedJob));
    unit_marks = take(batch * heads * row_blocks * rb / 16);
    part_marks = take(2 * kGroups * rb / 16);
    group_marks = take(kGroups * rb / 16);
    part_ml = take(2 * kGroups * rb * 2 * sizeof(float));
    part_o = take(2 * kGroups * rb * kValueDim * sizeof(float));
  }
  std::size_t rb, row_blocks, jobs, unit_marks, part_marks, group_marks, part_ml, part_o, bytes = 0;
};

template <int RT>
hipError_t launch_expanded(const ExpandedKernelArgs& k, const ExpandedStream& st, std::size_t units,
                           hipStream_t stream) {
  constexpr int RB = 64 * RT;
  const dim3 grid(static_cast<unsigned>(kGroups));
  expanded_kernel<4 * RT><<<grid, 256 * RT, 0, stream>>>(k, st);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  expanded_redo_kernel<RT><<<grid, 256, 0, stream>>>(k, st);
  e = hipGetLastError();
  if (e != hipSuccess) return e;
  const std::size_t rows = static_cast<std::size_t>(std::min(RB, k.tokens));
  const std::size_t jobs = st.by_unit != 0 ? units : kGroups;
  // Few units, so in many parts: workgroups of four rows.  (One head's 114 rows over
  // 7920 keys, twice: 39 us so, 107 with workgroups of 16 rows whose wavefronts have four
  // each.)
  const std::size_t wg_rows = units * kFewParts <= kGroups ? 4 : 16;
  const dim3 joins(static_cast<unsigned>(jobs), static_cast<unsigned>((rows + wg_rows - 1) / wg_rows));
  expanded_merge_kernel<<<joins, 256, 0, stream>>>(k, st, RB, static_cast<int>(wg_rows));
  return hipGetLastError();
}

}  // namespace

std::size_t expanded_workspace_bytes(std::size_t batch, std::size_t heads, std::size_t tokens,
                                     std::size_t) {
  return ExpandedLayout(batch, heads, tokens).bytes;
}

bool expanded_fits(const ExpandedArgs& a) {
  // Ranges, and places in them, are counted in 32 bits: of 2^38 tiles, a group's are
  // 2^30.
  const std::size_t units = a.batch * a.heads * ((a.tokens + 63) / 64);
  if (a.keys > 1 && std::max({a.key_at.token, a.rope_at.token, a.value_at.token}) >= kMostStride) {
    return false;
  }
  return units == 0 || a.keys / kTile + 2 + kStart <= (std::size_t{1} << 38) / units;
}

hipError_t launch_expanded_attention(const ExpandedArgs& a, hipStream_t stream) {
  if (a.batch == 0 || a.heads == 0 || a.tokens == 0) return hipSuccess;
  if (!expanded_fits(a)) return hipErrorInvalidValue;
  const ExpandedLayout layout(a.batch, a.heads, a.tokens);
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
  if (a.keys <= 1) k.key_at.token = k.rope_at.token = k.value_at.token = 0;
  k.qscale = kLog2e * a.scale;
  auto* const base = static_cast<unsigned char*>(a.workspace);
  ExpandedStream st{};
  st.jobs = reinterpret_cast<ExpandedJob*>(base + layout.jobs);
  st.unit_marks = base + layout.unit_marks;
  st.part_marks = base + layout.part_marks;
  st.group_marks = base + layout.group_marks;
  st.part_ml = reinterpret_cast<float*>(base + layout.part_ml);
  st.part_o = reinterpret_cast<float*>(base + layout.part_o);
  st.groups = static_cast<int>(kGroups);
  // Row blocks over a long history are about as long as each other, and read a key at
  // about one time where a range's units are of as many heads (4 x 32 heads, 512 rows
  // over 4096 keys: 553 us for 578, a third fewer reads past L2).  Those of a prompt
  // by itself grow, and so do their ranges' distances (64 heads, 2048 rows and keys:
  // 382 for 346).
  const std::size_t units = a.batch * a.heads * layout.row_blocks;
  st.by_unit = units <= kGroups ? 1 : 0;
  st.weave = a.keys / 2 < a.tokens
                 ? 1
                 : static_cast<int>(std::clamp<std::size_t>(units / kGroups, 1, a.heads));
  return layout.rb == 64 ? launch_expanded<1>(k, st, units, stream)
                         : launch_expanded<2>(k, st, units, stream);
}

}  // namespace helix::hip
