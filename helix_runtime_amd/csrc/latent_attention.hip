// Absorbed attention over a latent cache:
//
//   out_r = sum_j p_rj c_j[:L] / sum_j p_rj,  p_rj = exp(scale q_r . c_j - m_r),
//
// r over a sequence's query rows (heads times tokens), j over the tokens that row r
// sees, c_j the row of W = L + 64 elements that every head shares.
//
// Work split.  16 or 64 of a sequence's rows form a unit; one pass over the
// sequence's tokens serves them all.  A unit's tokens are tiles of 32 (fp32 pages:
// 16).  A row block's units of all sequences are a flat list of tiles (and of what units
// cost beside them), of which its share of a fixed grid of workgroups takes equal
// ranges, whatever the lengths; more than 32 row blocks have one list.  A unit
// inside one range is finished there; one that crosses ranges leaves a partial
// (maximum, sum, output) per range, which latent_merge_kernel joins.  A workgroup
// leaves at most two partials, its first unit's and its last one's, so the workspace
// depends on the grid, not on the batch.  Row blocks read the same pages at one time
// so, and as far as latent_share() says on one XCD.  (One sequence of 131071 tokens, 64
// rows in units of 16: 104 us with one list for all row blocks, 65 so.)
//
// Matrix form.  Per tile scores are S^T = C Q^T and outputs O^T += C^T P^T, a
// wavefront having 16 rows: a lane holds tokens of one query row, so a row's maximum
// takes two cross-lane steps and its probabilities are an operand as they are.  The
// tile lies in LDS once, and is read as rows for the scores and transposed for the
// outputs.  A wavefront's queries and outputs, 16 x W and 16 x L numbers, stay in its
// registers: 216 and 128 a lane, one wavefront a SIMD.  fp32 factors are sums of
// 16-bit terms, each product of terms exact in fp32:
// - bf16 pages: elements are one bf16 term, queries and probabilities three
//   (24 bits): 3 products;
// - fp8 pages: codes are exact in fp16, queries and probabilities two fp16 terms (22
//   bits and a sign: the rounding of an fp32 number): 2 products.  Terms must stay
//   above fp16's smallest numbers: a query row is scaled by a power of two that puts
//   its largest element in [2^10, 2^11), and probabilities (with them sums and
//   outputs) carry a factor of 2^8;
// - fp32 pages: the fp32 matrix instructions.
//
// What bounds it.  64 sequences of 512 to 8192 tokens, 16 heads, fp8 pages: 104 MB, 22
// us at a large copy's rate, 40 here, of which 12 are the start (the queries' way into
// registers, the first pages') and 8 the joins of wavefronts and of parts.  128 heads,
// bf16 pages: 54 Gflop, three times that in products, 133 us at the rate of a large
// bf16 matrix product, 148 here.  One sequence of 131071 tokens, 48 rows, bf16: 151
// MB, 32 us, 61 to 65 here.
//
// Units of 64 rows: four wavefronts with 16 rows each share a tile.  Units of 16 rows
// (what one token of 16 heads is): the wavefronts take tiles in turn, each by
// itself, and join what they have at the unit's end.  unit_rows() says which.
#include "bf16.hpp"
#include "fp8.hpp"
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
using prefill_detail::lds_address;
using prefill_detail::lds_load16_at;
using prefill_detail::row_max;
using prefill_detail::row_sum;
using prefill_detail::uniform_read;
using prefill_detail::v4f;
using prefill_detail::v4s;

typedef unsigned v2u __attribute__((ext_vector_type(2)));
typedef int v2i __attribute__((ext_vector_type(2)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef float v2f __attribute__((ext_vector_type(2)));
typedef __bf16 v2bf __attribute__((ext_vector_type(2)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr int P = static_cast<int>(kLatentPage);
constexpr int kWaves = 4;
// fp8 pages: the logarithm of the factor on probabilities.
constexpr float kProbLog = 8.0f;
// A row's reference stays while no score is above it by more than this (log2
// units): fp16's largest number is 2^16.
constexpr float kSlack = 7.0f;

struct LatentKernelArgs {
  const float* query;
  const void* pool;
  const std::uint32_t* tables;
  const std::int32_t* lengths;
  const std::int32_t* token_counts;
  float* out;
  Rows query_at, out_at;
  int batch, q_heads, tokens, max_blocks;
  int rows;  // query rows of a sequence: q_heads * tokens
  std::uint32_t physical_blocks;
  float qscale;  // log2(e) * scale, times the pages' scale
  float page_scale;
};

// A unit to join: the one that a group's range ends without starting it.
struct LatentJob {
  int b, rb;       // sequence (-1: none), row block
  int first, last; // groups whose ranges start and end the unit
};

struct LatentStream {
  float* part_o;   // [2 * groups, part_rows, L]
  float* part_ml;  // [2 * groups, part_rows, 2]
  int part_rows;   // a unit's rows, or 16 where there are no more
  LatentJob* jobs; // by unit where there are no more units than groups, else by group
  int groups;
  int row_blocks;  // units of a sequence
  int share;       // groups of a row block, or 0: none of its own
  int by_unit;
};

// The next term of x and y, rounded to nearest and packed into a word; x and y become
// what it leaves.
template <int PF>
__device__ __forceinline__ unsigned next_term(float& x, float& y) {
  if constexpr (PF == 2) {
    const v2h h = __builtin_convertvector((v2f{x, y}), v2h);
    x -= static_cast<float>(h[0]);
    y -= static_cast<float>(h[1]);
    return __builtin_bit_cast(unsigned, h);
  } else {
    const unsigned t = __builtin_bit_cast(unsigned, __builtin_convertvector((v2f{x, y}), v2bf));
    x -= __uint_as_float(t << 16);
    y -= __uint_as_float(t & 0xffff0000u);
    return t;
  }
}

// Four words of fp8 codes as fp16 are two of these.
__device__ __forceinline__ v4u codes_fp16(unsigned w0, unsigned w1) {
  return v4u{
      __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w0, 1.0f, false)),
      __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w0, 1.0f, true)),
      __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w1, 1.0f, false)),
      __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w1, 1.0f, true))};
}

// A tile in LDS: rows of kPitch bytes, whose 16-byte chunks are exchanged within
// groups of kMask + 1 by an exclusive or with `turn` of the row.  A read of a chunk of
// 16 rows (scores) and one of 16 dims of 4 or 8 rows (outputs) then hit distinct
// banks: 16-bit rows lie 1152 or 640 bytes apart, 128 from a multiple of 256, fp32 rows
// on one, and rows of codes 64 from one.  fp8 codes become fp16 on their way into LDS
// where four wavefronts read them (SHARED), else as they are read.
template <int PF, int L, bool SHARED>
struct Tile {
  static constexpr int W = L + static_cast<int>(kLatentRope);
  static constexpr bool kCodes = PF == 2 && !SHARED;
  static constexpr int kElem = PF == 0 ? 4 : kCodes ? 1 : 2;  // bytes in LDS
  static constexpr int kPageElem = PF == 0 ? 4 : PF == 1 ? 2 : 1;
  static constexpr int kTokens = PF == 0 ? 16 : 32;
  static constexpr int kPages = kTokens / P;
  static constexpr int kPitch = W * kElem;
  static constexpr int kBytes = kTokens * kPitch;
  static constexpr unsigned kMask = PF == 0 ? 15 : kCodes ? 3 : 7;
  // Loads of 16 bytes a lane (8, of codes that become fp16) come in kGroups groups of
  // kLoads, a group being kGroupRows whole rows.
  static constexpr int kLoads = W / 64;
  static constexpr int kGroups = kCodes ? 2 : 4;
  static constexpr int kGroupRows = kTokens / kGroups;
  static_assert(kGroups * kLoads * 1024 == kBytes && kGroupRows * kPitch == kLoads * 1024);
  static constexpr std::size_t kPageBytes = static_cast<std::size_t>(P) * W * kPageElem;
  static __device__ __forceinline__ unsigned turn(int row) {
    if constexpr (PF == 0) return static_cast<unsigned>(row & 15);
    if constexpr (kCodes) return static_cast<unsigned>(((row >> 2) & 3) ^ ((row >> 3) & 2));
    return static_cast<unsigned>(row & 6);
  }
};

// What a unit's start costs a workgroup that has begun with another one, in tiles: its
// queries have to come and be split, its first tiles are waited for, and the last
// unit's part joined and written.  (64 sequences of 512 to 8192 tokens, 16 heads, fp8
// pages: the slowest workgroup takes 52 us where starts count nothing, most take 30; the
// call takes 43 us with 12, 41 with 16, 38 with 24, 39 with 36.)
template <bool SHARED>
constexpr int start_cost() {
  return SHARED ? 4 : 24;
}

// A place in the flat list, in which each unit has start_cost() places before its
// tiles, and what of its unit is in the workgroup's range.
struct LatentCursor {
  int b, rb, blk, to;     // the next tile, and the end of the range's
  int left;               // places of the range behind the unit's
  long long base;         // the unit's first place
  int length, count, nb;  // the sequence's tokens, its query tokens, tiles
  int bad;                // its length lies outside its table
};

// Tiles of sequence b: one at least where it has rows.
template <int KT>
__device__ __forceinline__ int sequence_tiles(const LatentKernelArgs& a, int b) {
  if (b >= a.batch || clamped_count(a, b) == 0) return 0;
  const int length = a.lengths[b];
  if (length < 0 || length > a.max_blocks * P) return 1;
  return max((length + KT - 1) / KT, 1);
}

template <int KT>
__device__ __forceinline__ void load_sequence(const LatentKernelArgs& a, LatentCursor& c) {
  const int length = uniform_read(a.lengths + c.b);
  c.bad = length < 0 || length > a.max_blocks * P;
  c.length = c.bad ? 0 : length;
  c.count = a.tokens;
  if (a.token_counts != nullptr) c.count = min(max(uniform_read(a.token_counts + c.b), 0), a.tokens);
  c.nb = c.count > 0 ? max((c.length + KT - 1) / KT, 1) : 0;
}

// This group's first place, of ranges of `each` places; whether it has a tile.
template <int KT, int START, int LEAST>
__device__ __forceinline__ bool first_place(const LatentKernelArgs& a, const LatentStream& st,
                                            int group, int lane, long long& each, LatentCursor& c) {
  auto places = [&](int b) {
    const int nb = sequence_tiles<KT>(a, b);
    return nb > 0 ? nb + START : 0;
  };
  // Places of all sequences' units of one row block.
  const int mine = places(lane);
  const long long sums = lane_scan(mine, lane);
  long long per_block = uniform_long(__shfl(sums, 63, 64));
  if (a.batch > 64) {
    long long more = 0;
#pragma unroll 4
    for (int b0 = 64; b0 < a.batch; b0 += 64) more += places(b0 + lane);
    per_block += uniform_long(__shfl(lane_scan(more, lane), 63, 64));
  }
  // A row block's list to its share of the groups, or all of them to all.
  const int block = st.share > 0 ? group / st.share : 0;
  if (st.share > 0 && block >= st.row_blocks) return false;
  const int first_group = block * st.share;
  const long long total = st.share > 0 ? per_block : per_block * st.row_blocks;
  const int groups = st.share > 0 ? st.share : st.groups;
  each = divide(total + groups - 1, groups);
  each = uniform_long(max((each + LEAST - 1) / LEAST * LEAST, 1ll));
  const long long at = (group - first_group) * each;
  const long long have = min(each, total - at);
  if (have <= 0) return false;
  c.rb = __builtin_amdgcn_readfirstlane(block + static_cast<int>(divide(at, per_block)));
  const long long rem = at - (c.rb - block) * per_block;
  const long long g0 = group * each;
  long long base = 0;
  for (int b0 = 0; b0 < a.batch; b0 += 64) {
    const int n = b0 == 0 ? mine : places(b0 + lane);
    const long long sum = b0 == 0 ? sums : lane_scan(n, lane);
    const long long from = base + sum - n, to = base + sum;
    const unsigned long long hit = __ballot(from <= rem && rem < to);
    if (hit != 0) {
      const int src = __ffsll(static_cast<long long>(hit)) - 1;
      c.b = __builtin_amdgcn_readfirstlane(b0 + src);
      load_sequence<KT>(a, c);
      const int in = static_cast<int>(rem - uniform_long(__shfl(from, src, 64)));
      c.base = uniform_long(g0 - in);
      c.blk = __builtin_amdgcn_readfirstlane(max(in - START, 0));
      c.to = __builtin_amdgcn_readfirstlane(
          static_cast<int>(min(static_cast<long long>(c.nb), in + have - START)));
      c.left = __builtin_amdgcn_readfirstlane(
          static_cast<int>(max(have - (c.nb + START - in), 0ll)));
      break;
    }
    base += uniform_long(__shfl(sum, 63, 64));
  }
  return c.to > c.blk;
}

// Whether the range has tiles of a later unit, and that unit.
template <int START>
__device__ __forceinline__ bool more_units(const LatentCursor& c) {
  return c.left > START;
}
template <int KT, int START>
__device__ __forceinline__ void next_unit(const LatentKernelArgs& a, LatentCursor& c) {
  c.base += c.nb + START;
  do {
    if (++c.b == a.batch) {
      c.b = 0;
      ++c.rb;
    }
    load_sequence<KT>(a, c);
  } while (c.nb == 0);
  c.blk = 0;
  c.to = min(c.nb, c.left - START);
  c.left = max(c.left - c.nb - START, 0);
}

// One wavefront's 16 rows of a unit: queries, outputs, references and sums, and what
// a tile in LDS does to them.
template <int PF, int L, bool SHARED>
struct LatentRows {
  using T = Tile<PF, L, SHARED>;
  static constexpr int QT = PF == 0 ? 1 : PF == 1 ? 3 : 2;  // terms
  static constexpr int NS = PF == 0 ? T::W / 16 : T::W / 32;  // steps of the scores' sum
  static constexpr int ND = L / 16;                           // tiles of output dims
  static constexpr int NH = T::kTokens / 16;                  // 16-token halves

  v4u q[NS][QT];    // fp32 pages: four fp32 numbers
  v4f o[ND];        // o[dt][i]: dim 16 dt + 4 grp + i of row col
  float m, l;       // l: the lane's own tokens
  float unscale;    // fp8 pages: what undoes the row's power of two
  int limit;        // tokens that row col sees
  bool live;        // the row is one of the sequence's

  // Row r of the unit's sequence: its head and token.
  __device__ __forceinline__ void start(const LatentKernelArgs& a, const LatentCursor& c, int row,
                                        int grp) {
    live = row < a.rows;
    const int h = live ? row / a.tokens : 0;
    const int t = live ? row - h * a.tokens : 0;
    live = live && t < c.count;
    limit = c.length - c.count + t + 1;
    const float* const src = a.query + static_cast<std::size_t>(c.b) * a.query_at.batch +
                             static_cast<std::size_t>(h) * a.query_at.head +
                             static_cast<std::size_t>(t) * a.query_at.token;
    m = live ? -INFINITY : INFINITY;  // (a row that is none never moves the others)
    l = 0.f;
    // All of the row's loads at once.  (A row that is none reads the sequence's first
    // one; nothing of what comes of it is kept.)
    constexpr int NX = PF == 0 ? 1 : 2;
    v4f x[NS][NX];
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
      for (int w = 0; w < NX; ++w) {
        x[s][w] = *reinterpret_cast<const v4f*>(src + 16 * NX * s + 4 * NX * grp + 4 * w);
      }
    __builtin_amdgcn_sched_barrier(0);
    float grow = a.qscale;
    if constexpr (PF == 2) {
      float most = 0.f;
#pragma unroll
      for (int s = 0; s < NS; ++s)
#pragma unroll
        for (int w = 0; w < NX; ++w) {
          const v4f y = x[s][w];
          most = fmaxf(most, fmaxf(fmaxf(fabsf(y[0]), fabsf(y[1])), fmaxf(fabsf(y[2]), fabsf(y[3]))));
        }
      most = row_max(most);
      // most * 2^(10 - e) in [2^10, 2^11) for any number, or below for those of less than
      // 2^-110, as far as 2^(10 - e) is a normal number.
      const int e = min(max(static_cast<int>(__float_as_uint(most) >> 23) - 127, -110), 127);
      grow = __uint_as_float(static_cast<unsigned>(127 + 10 - e) << 23);
      unscale = __uint_as_float(static_cast<unsigned>(127 - 10 + e) << 23);
      // (Positive, or scores of -infinity would not stay that: the score scale's
      // sign goes with the queries, which a scale of 0 makes 0.)
      grow = a.qscale > 0.f ? grow : a.qscale < 0.f ? -grow : 0.f;
      unscale = fmaxf(unscale * fabsf(a.qscale), 1.2e-38f);
    }
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      if constexpr (PF == 0) {
        q[s][0] = __builtin_bit_cast(v4u, x[s][0] * grow);
      } else {
        unsigned w[4][3];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float y0 = x[s][i >> 1][2 * (i & 1)] * grow, y1 = x[s][i >> 1][2 * (i & 1) + 1] * grow;
#pragma unroll
          for (int n = 0; n < QT; ++n) w[i][n] = next_term<PF>(y0, y1);
        }
#pragma unroll
        for (int i = 0; i < QT; ++i) q[s][i] = v4u{w[0][i], w[1][i], w[2][i], w[3][i]};
      }
      keep(s);
    }
#pragma unroll
    for (int dt = 0; dt < ND; ++dt) o[dt] = v4f{0.f, 0.f, 0.f, 0.f};
  }

  // Half a wavefront's registers are accumulation registers, which matrix instructions
  // can take any operand from: the queries live there, everything else in the others.
  // (Said here, or the compiler mixes them and moves both to and fro.)
  __device__ __forceinline__ void keep(int s) {
#pragma unroll
    for (int i = 0; i < QT; ++i) asm("" : "+a"(q[s][i]));
  }

  // Scores of a tile: sc[h][i] is token 16 h + 4 grp + i of row col.  `beside(i)` is
  // what else the lane does behind the i-th of kSlots matrix instructions: one
  //  takes 16 cycles, of which its issue takes 4, and only what is issued
  // between two of them goes beside the first.
  static constexpr int kSlots = NS * (PF == 0 ? 1 : QT * NH);
  static constexpr bool kSpread = SHARED && PF != 0;  // a matrix instruction at a time
  template <typename F>
  __device__ __forceinline__ void scores(const unsigned char* tile, int col, int grp, v4f (&sc)[NH],
                                         F&& beside) const {
    constexpr int A = PF == 0 || T::kCodes ? 4 : 2;  // operands come out of LDS A steps ahead
    constexpr int AR = kSpread ? A + 1 : A;          // (kSpread: while the step's are in use)
    // Row col's chunk 4 s + grp (codes: half of chunk 2 s + grp / 2): its place within
    // a group of chunks is one of two (fp32 pages: four), by s.
    constexpr int V = PF == 0 ? 4 : 2;
    constexpr int C = T::kCodes ? 2 : 4;  // chunks of a step
    unsigned at[V][NH];
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
      for (int h = 0; h < NH; ++h) {
        const int row = 16 * h + col;
        const int chunk = C * i + (T::kCodes ? grp / 2 : grp);
        at[i][h] = static_cast<unsigned>(row * T::kPitch) +
                   ((static_cast<unsigned>(chunk) ^ T::turn(row)) & T::kMask) * 16u +
                   (T::kCodes ? (grp % 2) * 8u : 0u);
      }
    using Operand = std::conditional_t<T::kCodes, v2u, v4u>;
    Operand raw[AR][NH];
    auto read_half = [&](int s, int h) {
      raw[s % AR][h] = *reinterpret_cast<const Operand*>(tile + at[s % V][h] + (s / V) * (V * C * 16));
    };
    auto read = [&](int s) {
#pragma unroll
      for (int h = 0; h < NH; ++h) read_half(s, h);
    };
#pragma unroll
    for (int s = 0; s < A; ++s) read(s);
#pragma unroll
    for (int h = 0; h < NH; ++h) sc[h] = v4f{0.f, 0.f, 0.f, 0.f};
    [[maybe_unused]] v4f step_sum[2], low[NH];
#pragma unroll
    for (int h = 0; h < NH; ++h) low[h] = v4f{0.f, 0.f, 0.f, 0.f};
    // Codes become fp16 a step ahead, between the matrix instructions of the step.
    v4u wide[2][NH];
    auto widen = [&](int s) {
      if constexpr (T::kCodes) {
#pragma unroll
        for (int h = 0; h < NH; ++h) {
          wide[s % 2][h] = codes_fp16(raw[s % AR][h][0], raw[s % AR][h][1]);
        }
      }
    };
    widen(0);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      if constexpr (PF == 0) {
        const v4f x = __builtin_bit_cast(v4f, raw[s % AR][0]), y = __builtin_bit_cast(v4f, q[s][0]);
        // A step's sum by itself, and the last one's to the others': one sum of 576
        // products would be off by three times as much.
        v4f& sum = step_sum[s % 2];
        sum = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          sum = __builtin_amdgcn_mfma_f32_16x16x4f32(x[i], y[i], sum, 0, 0, 0);
        }
        if (s > 0) sc[0] += step_sum[(s + 1) % 2];
        if (s + 1 == NS) sc[0] += sum;
        beside(s);
      } else {
        v4u k[NH];
#pragma unroll
        for (int h = 0; h < NH; ++h) {
          if constexpr (T::kCodes) {
            k[h] = wide[s % 2][h];
          } else {
            k[h] = raw[s % AR][h];
          }
        }
        // Smallest products first.
#pragma unroll
        for (int i = QT - 1; i >= 0; --i) {
#pragma unroll
          for (int h = 0; h < NH; ++h) {
            // (Sums of the smaller terms' products by themselves: the rounding of the
            // larger ones' is then that of a third, or half, as many.)
            v4f& sum = i == 0 ? sc[h] : low[h];
            sum = matrix_step<PF == 2>(k[h], q[s][i], sum);
            const int at_step = NH * (QT - 1 - i) + h;
            if (kSpread && at_step % 2 == 1 && at_step / 2 < NH && s + A < NS) read_half(s + A, at_step / 2);
            if (kSpread || h == NH - 1) beside(NH * QT * s + at_step);
            if (kSpread) __builtin_amdgcn_sched_barrier(0);
          }
        }
      }
      if (s + 1 < NS) widen(s + 1);
      if (!kSpread && s + A < NS) read(s + A);
      __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (PF != 0) {
#pragma unroll
      for (int h = 0; h < NH; ++h) sc[h] += low[h];
    }
  }

  // A row's reference follows the tile's largest score where that is far above it.  (By
  // the row's own scores alone: no bit of it depends on another row's numbers, which may
  // be of tokens that it does not see, or of no query at all.)
  __device__ __forceinline__ void follow(const v4f (&sc)[NH]) {
    float mx = -INFINITY;
#pragma unroll
    for (int h = 0; h < NH; ++h) {
      mx = fmaxf(mx, fmaxf(fmaxf(sc[h][0], sc[h][1]), fmaxf(sc[h][2], sc[h][3])));
    }
    if constexpr (PF == 2) mx *= unscale;
    if (__ballot(mx > m + kSlack) != 0) {
      const float most = row_max(mx);
      const float mn = most > m + kSlack ? most : m;
      const float alpha = exp2_ratio(m, mn);
#pragma unroll
      for (int dt = 0; dt < ND; ++dt) {
        o[dt] *= alpha;
        if (dt % 4 == 3) __builtin_amdgcn_sched_barrier(0);
      }
      l *= alpha;
      m = mn;
    }
  }
  // What scores are taken relative to: rows that have seen nothing have no reference.
  __device__ __forceinline__ float reference() const {
    return (m == -INFINITY ? 0.f : m) - (PF == 2 ? kProbLog : 0.f);
  }

  // Probabilities of the scores as operands, in small parts: of two tokens an
  // exponential each, then a term of both each.
  static constexpr int kPairs = 2 * NH;
  static constexpr int kPartsOfPair = PF == 0 ? 1 : 2 + QT;
  static constexpr int kProbParts = kPairs * kPartsOfPair;
  struct Probabilities {
    unsigned w[kPairs][3];
    float f[PF == 0 ? 4 : 1];
    float y[2];  // what the terms so far leave
  };
  __device__ __forceinline__ void probability(int part, const v4f (&sc)[NH], float ref,
                                              Probabilities& p) {
    const int n = part / kPartsOfPair, level = part % kPartsOfPair;
    if (PF == 0 || level < 2) {
      const v4f x = sc[n / 2];
#pragma unroll
      for (int i = PF == 0 ? 0 : level; i < (PF == 0 ? 2 : level + 1); ++i) {
        const float s = x[2 * (n % 2) + i];
        if constexpr (PF == 2) {
          p.y[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s, unscale, -ref));
        } else {
          p.y[i] = __builtin_amdgcn_exp2f(s - ref);
        }
        if constexpr (PF == 0) p.f[2 * n + i] = p.y[i];
      }
      if constexpr (PF == 0) l += p.y[0] + p.y[1];
    } else {
      if (level == 2) l += p.y[0] + p.y[1];
      p.w[n][level - 2] = next_term<PF>(p.y[0], p.y[1]);
    }
  }
  // Outputs of the tile.
  __device__ __forceinline__ void add_values(const unsigned char* tile, int col, int grp,
                                             const Probabilities& p) {
    if constexpr (PF == 0) {
      constexpr int A = 4;
      // Token 4 grp + i's dim 16 dt + col, chunk 4 dt + col / 4.
      unsigned at[4][4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          const int row = 4 * grp + i;
          at[i][d] = static_cast<unsigned>(row * T::kPitch) +
                     ((static_cast<unsigned>(4 * d + (col >> 2)) ^ T::turn(row)) & T::kMask) * 16u +
                     (col & 3) * 4u;
        }
      float v[A][4];
      auto read = [&](int dt) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          v[dt % A][i] = *reinterpret_cast<const float*>(tile + at[i][dt % 4] + (dt / 4) * 256);
        }
      };
#pragma unroll
      for (int dt = 0; dt < A; ++dt) read(dt);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int dt = 0; dt < ND; ++dt) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          o[dt] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[dt % A][i], p.f[i], o[dt], 0, 0, 0);
        }
        if (dt + A < ND) read(dt + A);
        __builtin_amdgcn_sched_barrier(0);
      }
    } else {
      using LdsV4s = __attribute__((address_space(3))) v4s;
      constexpr int A = T::kCodes ? 6 : 4;
      constexpr int AR = kSpread ? A + 2 : A;
      v4u pop[QT];
#pragma unroll
      for (int i = 0; i < QT; ++i) pop[i] = v4u{p.w[0][i], p.w[1][i], p.w[2][i], p.w[3][i]};
      // 16 dims of tokens 4 grp .. + 3 and 16 + 4 grp .. + 3: 32 bytes a token, which
      // four lanes read (codes: 16 bytes, two lanes), and each lane gets a dim.
      using LdsV2i = __attribute__((address_space(3))) v2i;
      constexpr int V = 4;
      const int row = T::kCodes ? 4 * grp + ((col >> 1) & 3) + 2 * (col & 8) : 4 * grp + (col >> 2);
      unsigned at[V];
#pragma unroll
      for (int d = 0; d < V; ++d) {
        const int chunk = T::kCodes ? d : 2 * d + ((col >> 1) & 1);
        at[d] = static_cast<unsigned>(row * T::kPitch) +
                ((static_cast<unsigned>(chunk) ^ T::turn(row)) & T::kMask) * 16u + (col & 1) * 8u;
      }
      using Operand = std::conditional_t<T::kCodes, v2i, v4u>;
      Operand raw[AR];
      // Tokens 4 grp and on, then (part 1) those 16 behind them.
      auto read_part = [&](int dt, int part) {
        const unsigned char* const from = tile + at[dt % V] + (dt / V) * (T::kCodes ? 64 : 128);
        if constexpr (T::kCodes) {
          if (part == 0) raw[dt % AR] = __builtin_amdgcn_ds_read_tr8_b64_v2i32((LdsV2i*)(from));
        } else {
          const v4s x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsV4s*)(from + part * 16 * T::kPitch));
          const v2u y = __builtin_bit_cast(v2u, x);
          raw[dt % AR][2 * part] = y[0];
          raw[dt % AR][2 * part + 1] = y[1];
        }
      };
      auto read = [&](int dt) {
        read_part(dt, 0);
        read_part(dt, 1);
      };
#pragma unroll
      for (int dt = 0; dt < A; ++dt) read(dt);
      v4u wide[4];
      auto widen = [&](int dt) {
        if constexpr (T::kCodes) {
#pragma unroll
          for (int d = dt; d < dt + 2; ++d) {
            wide[d % 4] = codes_fp16(static_cast<unsigned>(raw[d % AR][0]),
                                     static_cast<unsigned>(raw[d % AR][1]));
          }
        }
      };
      widen(0);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int dt = 0; dt < ND; dt += 2) {
        v4u v[2];
#pragma unroll
        for (int d = 0; d < 2; ++d) {
          if constexpr (T::kCodes) {
            v[d] = wide[(dt + d) % 4];
          } else {
            v[d] = raw[(dt + d) % AR];
          }
        }
#pragma unroll
        for (int i = QT - 1; i >= 0; --i)
#pragma unroll
          for (int d = 0; d < 2; ++d) {
            o[dt + d] = matrix_step<PF == 2>(v[d], pop[i], o[dt + d]);
            const int at_step = 2 * (QT - 1 - i) + d;
            if (kSpread && at_step < 4 && dt + A < ND) read_part(dt + A + at_step / 2, at_step % 2);
            if (kSpread) __builtin_amdgcn_sched_barrier(0);
          }
        if (dt + 2 < ND) widen(dt + 2);
        if (!kSpread && dt + A < ND) {
          read(dt + A);
          read(dt + A + 1);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  }

  // Scores of a tile whose first token is `first`: those that the row does not see
  // become -infinity, and NaN where `poison` (bit: token of the tile) has one it sees.
  __device__ __forceinline__ void mask(int first, unsigned poison, int grp, v4f (&sc)[NH]) const {
#pragma unroll
    for (int h = 0; h < NH; ++h)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int n = 16 * h + 4 * grp + i;
        float x = sc[h][i];
        if (((poison >> n) & 1u) != 0) x = NAN;
        sc[h][i] = first + n < limit ? x : -INFINITY;
      }
  }
};

// Where the pages' elements of a tile come from, and their way into LDS.
template <int PF, int L, bool SHARED>
struct TileLoader {
  using T = Tile<PF, L, SHARED>;
  static constexpr bool kConvert = PF == 2 && SHARED;
  unsigned off[T::kLoads];  // of the lane's bytes in a group of rows

  __device__ __forceinline__ void start(int lane) {
#pragma unroll
    for (int i = 0; i < T::kLoads; ++i) {
      const unsigned o = static_cast<unsigned>(i * 1024 + lane * 16);
      const unsigned row = o / T::kPitch, c = (o - row * T::kPitch) / 16;
      const unsigned from = c ^ (T::turn(static_cast<int>(row)) & T::kMask);
      off[i] = (row * T::kPitch + from * 16) / (kConvert ? 2 : 1);
    }
  }
  // Group g's rows lie in page g / (groups of a page); their turns differ from the
  // first group's by one exchange.
  static constexpr int kPageGroups = P / T::kGroupRows;
  static __device__ __forceinline__ unsigned exchange(int g) {
    return PF == 0 ? 64u * g : T::kCodes ? 32u * g : 0u;
  }
  static __device__ __forceinline__ const unsigned char* group_base(const unsigned char* page,
                                                                    int g) {
    return page + (g % kPageGroups) * (T::kGroupRows * T::W * T::kPageElem);
  }
  // Straight into LDS.
  __device__ __forceinline__ void direct(const unsigned char* page, int g, unsigned lds) const {
#pragma unroll
    for (int i = 0; i < T::kLoads; ++i) direct(page, g, lds, i);
  }
  __device__ __forceinline__ void direct(const unsigned char* page, int g, unsigned lds, int i) const {
    lds_load16_at(group_base(page, g), off[i] ^ exchange(g), lds + (g * T::kLoads + i) * 1024u);
  }
  // Codes into registers, and from there as fp16 into LDS.
  __device__ __forceinline__ void fetch(const unsigned char* page, int g, v2u (&raw)[T::kLoads]) const {
    using Global = const __attribute__((address_space(1))) v2u*;
    using GlobalBytes = const __attribute__((address_space(1))) unsigned char*;
    const auto base = reinterpret_cast<GlobalBytes>(
        reinterpret_cast<std::uintptr_t>(group_base(page, g)));
#pragma unroll
    for (int i = 0; i < T::kLoads; ++i) {
      raw[i] = __builtin_nontemporal_load(reinterpret_cast<Global>(base + (off[i] ^ exchange(g))));
    }
  }
  static __device__ __forceinline__ void store(unsigned char* tile, int g, int lane,
                                               const v2u (&raw)[T::kLoads]) {
#pragma unroll
    for (int i = 0; i < T::kLoads; ++i) {
      *reinterpret_cast<v4u*>(tile + (g * T::kLoads + i) * 1024 + lane * 16) =
          codes_fp16(raw[i][0], raw[i][1]);
    }
  }
};

// Rows of the tile that not all of a unit's query rows see must be finite: those
// behind the sequence's last become 0, and of the step's own tokens those that are
// not finite; the latter's bits are returned.  Rows 4 `wave` and on by 16 (4 rows at a
// time, 16 lanes each).
template <int PF, int L, bool SHARED>
__device__ __forceinline__ unsigned clean_rows(unsigned char* tile, int first, int from, int length,
                                               int lane, int row0, int row_step) {
  using T = Tile<PF, L, SHARED>;
  unsigned poison = 0;
  for (int r = row0 + (lane >> 4); r < T::kTokens; r += row_step) {
    unsigned char* const row = tile + r * T::kPitch;
    const int token = first + r;
    bool wipe = token >= length;
    if (!wipe && token >= from) {
      unsigned all = 0;  // bit 0: an element that is not finite
      for (int c = lane & 15; c < T::kPitch / 16; c += 16) {
        const v4u x = *reinterpret_cast<const v4u*>(row + c * 16);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if constexpr (PF == 0) {
            all |= (x[i] & 0x7f800000u) == 0x7f800000u;
          } else if constexpr (T::kCodes) {
            all |= (((x[i] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) != 0;
          } else {
            constexpr unsigned e = PF == 1 ? 0x7f80u : 0x7c00u;
            all |= (x[i] & e) == e || ((x[i] >> 16) & e) == e;
          }
        }
      }
      const unsigned long long hit = __ballot(all != 0);
      wipe = ((hit >> (lane & 48)) & 0xffffull) != 0;
      if (wipe) poison |= 1u << r;
    }
    if (wipe) {
      for (int c = lane & 15; c < T::kPitch / 16; c += 16) {
        *reinterpret_cast<v4u*>(row + c * 16) = v4u{0u, 0u, 0u, 0u};
      }
    }
  }
  return poison;
}

template <int PF, int L, bool SHARED>
struct LatentShared {
  using T = Tile<PF, L, SHARED>;
  // A wavefront by itself has one tile, or two of codes.
  static constexpr int kRing = T::kCodes ? 2 : 1;
  static constexpr int kBuffers = SHARED ? (PF == 2 ? 3 : 4) : kWaves;
  __align__(1024) unsigned char tile[kBuffers][(SHARED ? 1 : kRing) * T::kBytes];
  float ml[kWaves][16][2];
  unsigned poison[kWaves];
};

template <int PF, int L>
__device__ __forceinline__ float finish_factor(const LatentKernelArgs& a, bool complete, bool bad,
                                               float sum, bool some) {
  const float f = PF == 2 ? a.page_scale : 1.0f;
  if (!complete) return f;
  return bad ? NAN : row_factor(sum, some, f);
}

template <int PF, int L, bool SHARED>
__device__ __forceinline__ void latent_body(const LatentKernelArgs& a, const LatentStream& st,
                                            LatentShared<PF, L, SHARED>& sh) {
  using T = Tile<PF, L, SHARED>;
  using R = LatentRows<PF, L, SHARED>;
  using Loader = TileLoader<PF, L, SHARED>;
  constexpr int KT = T::kTokens;
  constexpr int RB = SHARED ? 16 * kWaves : 16;
  constexpr int NH = R::NH;
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, grp = lane >> 4;
  const int group = static_cast<int>(blockIdx.x);
  auto barrier = [] {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };
  if (st.by_unit == 0 && tid == 0) st.jobs[group] = LatentJob{-1, 0, 0, 0};
  constexpr int START = start_cost<SHARED>();
  LatentCursor cur{};
  long long each;
  // (Four wavefronts take tiles in turn: ranges of whole turns.)
  if (!first_place<KT, START, SHARED ? 1 : kWaves>(a, st, group, lane, each, cur)) return;

  Loader loader;
  loader.start(lane);
  const auto* const pool = static_cast<const unsigned char*>(a.pool);
  // The pages of a sequence being loaded, 64 at a time: lane i holds page pages_at + i
  // of pages_of.  Behind its tokens the last page is read again, and without tokens,
  // or where a page is none, page 0; what is read there takes no part.
  unsigned page_lane = 0;
  int pages_of = -1, pages_at = 0, bad_page = 0;
  struct Pages {
    const unsigned char* at[T::kPages];
    int bad;
  };
  auto locate = [&](const LatentCursor& c, int blk) {
    Pages p{};
    int first = blk * T::kPages - pages_at;
    if (__builtin_expect(pages_of != c.b || first < 0 || first + T::kPages > 64, 0)) {
      pages_of = c.b;
      pages_at = blk * T::kPages;
      first = 0;
      page_lane = 0;
      bad_page = c.bad;
      if (c.length > 0) {
        page_lane = a.tables[static_cast<std::size_t>(c.b) * a.max_blocks +
                             min(pages_at + lane, (c.length - 1) / P)];
        const bool outside = page_lane >= a.physical_blocks;
        if (__ballot(outside) != 0) bad_page = 1;
        if (outside) page_lane = 0;
      }
    }
    p.bad = bad_page;
#pragma unroll
    for (int i = 0; i < T::kPages; ++i) {
      p.at[i] = pool + static_cast<unsigned>(__builtin_amdgcn_readlane(page_lane, first + i)) *
                           T::kPageBytes;
    }
    return p;
  };
  auto page_of = [&](const Pages& p, int g) {
    if constexpr (T::kPages == 1) {
      return p.at[0];
    } else {
      return g < Loader::kPageGroups ? p.at[0] : p.at[1];
    }
  };

  R rows;
  // Ends the unit's part, tiles [from, c.to) of it.
  auto part_of = [&](const LatentCursor& c, int from) {
    const bool starts = from == 0, ends = c.to == c.nb;
    const int slot = 2 * group + (starts ? 1 : 0);
    if (ends && tid == 0) {
      const long long first = divide(c.base + START, each);
      if (st.by_unit != 0) {
        st.jobs[static_cast<std::size_t>(c.rb) * a.batch + c.b] =
            LatentJob{starts ? -1 : c.b, c.rb, static_cast<int>(first), group};
      } else if (!starts) {
        st.jobs[group] = LatentJob{c.b, c.rb, static_cast<int>(first), group};
      }
    }
    return slot;
  };
  // Row `row` of the sequence, dims `at` and on of its output or partial.
  auto out_row = [&](const LatentCursor& c, int row) {
    const int h = row / a.tokens, t = row - h * a.tokens;
    return a.out + static_cast<std::size_t>(c.b) * a.out_at.batch +
           static_cast<std::size_t>(h) * a.out_at.head + static_cast<std::size_t>(t) * a.out_at.token;
  };

  if constexpr (SHARED) {
    constexpr int NB = LatentShared<PF, L, SHARED>::kBuffers;
    const unsigned lds0 = lds_address(sh.tile[0]);
    // Tile i of the range goes to buffer i % NB, two steps (fp8: one step and the
    // registers) ahead of its scores.  Behind the range the last one is read again.
    LatentCursor ahead = cur;
    int located = 0;  // the range's tile that `next` is
    unsigned bads = 0;  // bit i % 32: of tile i
    v2u raw[PF == 2 ? T::kLoads : 1];
    Pages next = locate(ahead, ahead.blk);
    bads = next.bad != 0 ? 1u : 0u;
    auto locate_next = [&] {
      if (ahead.blk + 1 < ahead.to || more_units<START>(ahead)) {
        ++located;
        if (++ahead.blk == ahead.to) next_unit<KT, START>(a, ahead);
        next = locate(ahead, ahead.blk);
        bads = (bads & ~(1u << (located & 31))) | (next.bad != 0 ? 1u << (located & 31) : 0u);
      }
    };
    int into = 0;
    auto bump = [&](int& i) { i = i + 1 == NB ? 0 : i + 1; };
    // The wavefront's quarter of the next tile is sent for (fp8: the one that was
    // goes to LDS first), a load at a time.
    auto send = [&](int i) {
      if constexpr (PF == 2) {
        if (i != 0) return;
        Loader::store(sh.tile[into], wave, lane, raw);
        loader.fetch(page_of(next, wave), wave, raw);
      } else {
        loader.direct(page_of(next, wave), wave, lds0 + static_cast<unsigned>(into) * T::kBytes, i);
      }
    };
    auto sent = [&] {
      bump(into);
      locate_next();
    };
    auto send_all = [&] {
#pragma unroll
      for (int i = 0; i < T::kLoads; ++i) send(i);
      sent();
    };
    // What was sent for before the last two times is there.
    auto arrived = [&] {
      if constexpr (PF != 2) __builtin_amdgcn_s_waitcnt(0x0f70 | T::kLoads);
    };
    if constexpr (PF == 2) {
      loader.fetch(page_of(next, wave), wave, raw);
      locate_next();
    }
    send_all();
    send_all();
    if constexpr (PF != 2) send_all();
    arrived();
    barrier();
    int n = 0, buf = 0;  // tile, and its buffer
    for (;;) {
      const int row = cur.rb * RB + wave * 16 + col;
      rows.start(a, cur, row, grp);
      const int from = cur.blk, to = cur.to;
      // Tiles before `whole` are seen by every row.
      const int whole = max(cur.length - cur.count + 1, 0) / KT;
      int bad = 0;
      v4f sc[NH];
      rows.scores(sh.tile[buf], col, grp, sc, [](int) {});
      for (int blk = from; blk < to; ++blk) {
        if constexpr (PF == 2) send(0);
        bad |= static_cast<int>(bads >> (n & 31)) & 1;
        typename R::Probabilities p;
        int after = buf;
        bump(after);
        if (blk >= whole) {
          unsigned poison = clean_rows<PF, L, SHARED>(sh.tile[buf], blk * KT, cur.length - cur.count + 1,
                                              cur.length, lane, 4 * wave, 16);
#pragma unroll
          for (int bit = 16; bit < 64; bit *= 2) poison |= __shfl_xor(poison, bit, 64);
          if (lane == 0) sh.poison[wave] = poison;
          // (Of a unit's first tile other wavefronts may be taking scores still: those of
          // rows that are wiped meanwhile are ones that mask() replaces.)
          barrier();
          poison = sh.poison[0] | sh.poison[1] | sh.poison[2] | sh.poison[3];
          rows.mask(blk * KT, poison, grp, sc);
        }
        rows.follow(sc);
        const float ref = rows.reference();
        if (blk + 1 < to) {
          // This tile's probabilities beside the next one's scores.
          v4f now[NH];
#pragma unroll
          for (int h = 0; h < NH; ++h) now[h] = sc[h];
          constexpr int kApart = (R::kSlots - R::kProbParts) / T::kLoads;
          static_assert(kApart > 0, "a slot a part");
          // (A copy that the compiler does not know, or it takes the exponentials of
          // both cases out in front.)
          float ref_here = ref;
          asm("" : "+v"(ref_here));
          rows.scores(sh.tile[after], col, grp, sc, [&](int i) {
            if (i < R::kProbParts) rows.probability(i, now, ref_here, p);
            const int j = i - R::kProbParts;
            if (PF != 2 && j >= 0 && j % kApart == 0 && j / kApart < T::kLoads) send(j / kApart);
          });
        } else {
#pragma unroll
          for (int i = 0; i < R::kProbParts; ++i) rows.probability(i, sc, ref, p);
          if constexpr (PF != 2) {
#pragma unroll
            for (int i = 0; i < T::kLoads; ++i) send(i);
          }
        }
        sent();
        rows.add_values(sh.tile[buf], col, grp, p);
        buf = after;
        ++n;
        arrived();
        barrier();
      }
      // The part's end.
      const bool complete = from == 0 && to == cur.nb;
      const int slot = part_of(cur, from);
      const float sum = row_sum(rows.l);
      const bool some = from * KT < rows.limit;  // of the part's tokens
      const float f = finish_factor<PF, L>(a, complete, bad != 0, sum, some);
      if (rows.live) {
        const int local = wave * 16 + col;
        float* const dst = (complete ? out_row(cur, row)
                                     : st.part_o + (static_cast<std::size_t>(slot) * st.part_rows + local) * L) +
                           4 * grp;
#pragma unroll
        for (int dt = 0; dt < R::ND; ++dt) *reinterpret_cast<v4f*>(dst + 16 * dt) = rows.o[dt] * f;
        if (!complete && grp == 0) {
          float* const ml = st.part_ml + (static_cast<std::size_t>(slot) * st.part_rows + local) * 2;
          ml[0] = sum == 0.f && some ? kNoWeights : rows.m;
          ml[1] = bad != 0 ? NAN : sum;
        }
      }
      if (!more_units<START>(cur)) break;
      next_unit<KT, START>(a, cur);
    }
    // (Nothing is on its way into LDS when the workgroup gives it back.)
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  } else {
    constexpr int kRing = LatentShared<PF, L, SHARED>::kRing;
    unsigned char* const own_tiles = sh.tile[wave];
    const unsigned lds = lds_address(own_tiles);
    for (;;) {
      const int row = cur.rb * RB + col;
      const int from = cur.blk, to = cur.to;
      const int whole = max(cur.length - cur.count + 1, 0) / KT;
      int bad = 0;
      // The wavefront's i-th tile of the part into its place.
      auto send = [&](int i) {
        const int blk = from + wave + i * kWaves;
        if (blk >= to) return;
        const Pages p = locate(cur, blk);
        bad |= p.bad;
        const unsigned into = lds + static_cast<unsigned>(i % kRing) * T::kBytes;
#pragma unroll
        for (int g = 0; g < T::kGroups; ++g) loader.direct(page_of(p, g), g, into);
      };
#pragma unroll
      for (int i = 0; i < kRing; ++i) send(i);
      rows.start(a, cur, row, grp);
      for (int i = 0; from + wave + i * kWaves < to; ++i) {
        const int blk = from + wave + i * kWaves;
        if (kRing > 1 && blk + kWaves < to) {  // the next tile is on its way behind it
          asm volatile("s_waitcnt vmcnt(%0)" ::"n"(T::kGroups * T::kLoads) : "memory");
        } else {
          asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        }
        unsigned char* const tile = own_tiles + (i % kRing) * T::kBytes;
        v4f sc[NH];
        rows.scores(tile, col, grp, sc, [](int) {});
        if (blk >= whole) {
          unsigned poison = clean_rows<PF, L, SHARED>(tile, blk * KT, cur.length - cur.count + 1,
                                                      cur.length, lane, 0, 4);
#pragma unroll
          for (int bit = 16; bit < 64; bit *= 2) poison |= __shfl_xor(poison, bit, 64);
          rows.mask(blk * KT, poison, grp, sc);
        }
        rows.follow(sc);
        const float ref = rows.reference();
        typename R::Probabilities p;
#pragma unroll
        for (int j = 0; j < R::kProbParts; ++j) rows.probability(j, sc, ref, p);
        rows.add_values(tile, col, grp, p);
        // (The tile's reads are done before it is written again.)
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        send(i + kRing);
      }
      unsigned char* const tile = own_tiles;
      // The wavefronts join what they have: each one's outputs, relative to the
      // largest reference, in its tile.
      const float own = row_sum(rows.l);
      if (grp == 0) {
        sh.ml[wave][col][0] = rows.m;
        sh.ml[wave][col][1] = own;
      }
      if (lane == 0) sh.poison[wave] = static_cast<unsigned>(bad);
      barrier();
      float top = sh.ml[0][col][0];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) top = fmaxf(top, sh.ml[w][col][0]);
      float sum = 0.f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        // (A reference of -infinity comes with a sum of 0.)
        const float x = sh.ml[w][col][1];
        sum += x == 0.f ? 0.f : x * exp2_ratio(sh.ml[w][col][0], top);
      }
      bad = static_cast<int>(sh.poison[0] | sh.poison[1] | sh.poison[2] | sh.poison[3]);
      const float alpha = exp2_ratio(rows.m, top);
      // Row col's dims 4 u .. + 3 at chunk u ^ (col / 2 and 1 bit), 16 bytes each: the
      // 16 rows of one write, or read, lie on distinct banks.
      constexpr int kRowBytes = L * 4;
      auto place = [&](int r, int u) { return r * kRowBytes + ((u ^ r) & 15) * 16 + (u & ~15) * 16; };
#pragma unroll
      for (int dt = 0; dt < R::ND; ++dt) {
        *reinterpret_cast<v4f*>(tile + place(col, 4 * dt + grp)) = rows.o[dt] * alpha;
      }
      barrier();
      const bool complete = from == 0 && to == cur.nb;
      const int slot = part_of(cur, from);
      const bool some = from * KT < rows.limit;  // of the part's tokens
      const float f = finish_factor<PF, L>(a, complete, bad != 0, sum, some);
      if (sum == 0.f && some) top = kNoWeights;
      // A wavefront adds up four rows, 16 lanes (L / 16 dims each) a row.
      {
        const int local = 4 * wave + grp;
        const int r = cur.rb * RB + local;
        const float rf = __shfl(f, local, 64);
        const float rm = __shfl(top, local, 64), rs = __shfl(sum, local, 64);
        const bool live = __shfl(rows.live ? 1 : 0, local, 64) != 0;
        if (live) {
          float* const dst = complete
                                 ? out_row(cur, r)
                                 : st.part_o + (static_cast<std::size_t>(slot) * st.part_rows + local) * L;
#pragma unroll
          for (int i = 0; i < L / 64; ++i) {
            const int u = 16 * i + col;
            v4f x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
              x += *reinterpret_cast<const v4f*>(sh.tile[w] + place(local, u));
            }
            *reinterpret_cast<v4f*>(dst + 4 * u) = x * rf;
          }
          if (!complete && col == 0) {
            float* const ml = st.part_ml + (static_cast<std::size_t>(slot) * st.part_rows + local) * 2;
            ml[0] = rm;
            ml[1] = bad != 0 ? NAN : rs;
          }
        }
      }
      if (!more_units<START>(cur)) break;
      next_unit<KT, START>(a, cur);
      barrier();  // the tiles are read
    }
  }
}

template <int PF, int L, bool SHARED>
__global__ __launch_bounds__(64 * kWaves) __attribute__((amdgpu_waves_per_eu(1, 1)))
    void latent_kernel(LatentKernelArgs a, LatentStream st) {
  __shared__ LatentShared<PF, L, SHARED> sh;
  latent_body<PF, L, SHARED>(a, st, sh);
}

// Joins the partials of the units that cross ranges: the first group's second slot
// and the later groups' first ones.  blockIdx.x is a unit or a group.
constexpr int kMostParts = 512;
struct MergeRow {
  int row, h, t;
  bool live;
};
__device__ __forceinline__ MergeRow merge_row(const LatentKernelArgs& a, const LatentJob& job,
                                              int rb_rows, int local) {
  MergeRow r;
  r.row = job.rb * rb_rows + local;
  r.h = r.row / a.tokens;
  r.t = r.row - r.h * a.tokens;
  r.live = local < rb_rows && r.row < a.rows && r.t < clamped_count(a, job.b);
  return r;
}
__device__ __forceinline__ std::size_t merge_slot(const LatentJob& job, int part_rows, int local, int i) {
  return static_cast<std::size_t>(2 * (job.first + i) + (i == 0 ? 1 : 0)) * part_rows + local;
}
__device__ __forceinline__ float* merge_out(const LatentKernelArgs& a, const LatentJob& job,
                                            const MergeRow& r) {
  return a.out + static_cast<std::size_t>(job.b) * a.out_at.batch +
         static_cast<std::size_t>(r.h) * a.out_at.head + static_cast<std::size_t>(r.t) * a.out_at.token;
}

// Units in few parts: a wavefront has one of the four rows of blockIdx.y.  Where a unit
// has many all the same, the four share each row's.  (64 sequences of 4096 tokens, 16
// rows, bf16 pages: 68 us with their join this way, 79 the other; one of 131071 tokens,
// 32 rows: 110 this way, 62 the other.)
constexpr int kFewParts = 16;
template <int L>
__global__ __launch_bounds__(256) void latent_merge_kernel(LatentKernelArgs a, LatentStream st,
                                                           int rb_rows) {
  constexpr int NV = L / 256;  // 4 dims each
  constexpr int U = 4;         // partials on their way
  __shared__ float weights[4][kMostParts];
  __shared__ v4f sums[4][L / 4];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  if (st.by_unit != 0 && clamped_count(a, static_cast<int>(blockIdx.x) % a.batch) == 0) return;
  const LatentJob job = st.jobs[blockIdx.x];
  if (job.b < 0) return;
  const int local0 = static_cast<int>(blockIdx.y) * 4, local = local0 + wave;
  const MergeRow r = merge_row(a, job, rb_rows, local);
  const int parts = min(job.last - job.first + 1, kMostParts);
  // Partials `first`, first + step, .. of row local0 + w on their way.
  using Parts = v4f[U][NV];
  auto load = [&](int w, int first, int step, Parts& x) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = min(first + u * step, parts - 1);
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        x[u][v] = reinterpret_cast<const v4f*>(
            st.part_o + merge_slot(job, st.part_rows, local0 + w, i) * L)[64 * v + lane];
      }
    }
  };
  // The first ones are sent for before their weights are known.
  Parts begun;
  const int first = parts <= kFewParts ? 0 : wave, step = parts <= kFewParts ? 1 : 4;
  if (r.live && parts <= kFewParts) load(wave, first, step, begun);
  float top = -INFINITY, sum = 0.f;
  if (r.live) {
    for (int i0 = 0; i0 < parts; i0 += 64) {
      const int i = i0 + lane;
      v2f ml = {-INFINITY, 0.f};
      if (i < parts) {
        ml = *reinterpret_cast<const v2f*>(st.part_ml + 2 * merge_slot(job, st.part_rows, local, i));
      }
      float most = ml[0];
#pragma unroll
      for (int k = 32; k > 0; k /= 2) most = fmaxf(most, __shfl_xor(most, k, 64));
      // (Weights so far are relative to the largest so far.)
      const float now = fmaxf(top, most);
      const float turn = exp2_ratio(top, now);
      if (turn != 1.f) {
        for (int j = lane; j < i0; j += 64) weights[wave][j] *= turn;
      }
      const float f = ml[1] == 0.f ? 0.f : exp2_ratio(ml[0], now);
      if (i < parts) weights[wave][i] = f;
      float add = ml[1] * f;
#pragma unroll
      for (int k = 32; k > 0; k /= 2) add += __shfl_xor(add, k, 64);
      sum = sum * turn + add;
      top = now;
    }
  }
  // Of row local0 + w, partials first, first + step, ..; the first U are in x.
  auto gather = [&](int w, Parts& x, v4f (&o)[NV]) {
#pragma unroll
    for (int v = 0; v < NV; ++v) o[v] = v4f{0.f, 0.f, 0.f, 0.f};
    for (int i0 = first; i0 < parts; i0 += U * step) {
      if (i0 != first) load(w, i0, step, x);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = i0 + u * step;
        const float f = i < parts ? weights[w][min(i, parts - 1)] : 0.f;
        if (f != 0.f) {  // (a part that saw nothing has no outputs to speak of)
#pragma unroll
          for (int v = 0; v < NV; ++v) o[v] += x[u][v] * f;
        }
      }
    }
  };
  v4f o[NV];
  if (parts <= kFewParts) {
    if (r.live) gather(wave, begun, o);
  } else {
    for (int w = 0; w < 4; ++w) {
      __syncthreads();
      if (!merge_row(a, job, rb_rows, local0 + w).live) continue;
      v4f own[NV];
      load(w, first, step, begun);
      gather(w, begun, own);
#pragma unroll
      for (int v = 0; v < NV; ++v) sums[wave][64 * v + lane] = own[v];
      __syncthreads();
      if (wave != w) continue;
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        o[v] = sums[0][64 * v + lane];
#pragma unroll
        for (int k = 1; k < 4; ++k) o[v] += sums[k][64 * v + lane];
      }
    }
  }
  if (!r.live) return;
  const float f = row_factor(sum, top != -INFINITY, 1.0f);
  auto* const dst = reinterpret_cast<v4f*>(merge_out(a, job, r));
#pragma unroll
  for (int v = 0; v < NV; ++v) dst[64 * v + lane] = o[v] * f;
}

// Few units in many parts: a workgroup has 128 dims (blockIdx.z) of a row (blockIdx.y),
// each half of its eight wavefronts every 16th partial.
constexpr int kSplitDims = 128;
template <int L>
__global__ __launch_bounds__(512) void latent_split_merge_kernel(LatentKernelArgs a, LatentStream st,
                                                                 int rb_rows) {
  constexpr int kShares = 16, U = 8;
  __shared__ float weights[kMostParts];
  __shared__ float lead[8], total[8];
  __shared__ v4f sums[kShares][kSplitDims / 4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  if (st.by_unit != 0 && clamped_count(a, static_cast<int>(blockIdx.x) % a.batch) == 0) return;
  const LatentJob job = st.jobs[blockIdx.x];
  if (job.b < 0) return;
  const int local = static_cast<int>(blockIdx.y);
  const MergeRow r = merge_row(a, job, rb_rows, local);
  if (!r.live) return;
  const int parts = min(job.last - job.first + 1, kMostParts);
  // A thread has a partial's maximum and sum.
  float pm = -INFINITY, pl = 0.f;
  if (tid < parts) {
    const float* const ml = st.part_ml + 2 * merge_slot(job, st.part_rows, local, tid);
    pm = ml[0];
    pl = ml[1];
  }
  float top = pm;
#pragma unroll
  for (int k = 32; k > 0; k /= 2) top = fmaxf(top, __shfl_xor(top, k, 64));
  if (lane == 0) lead[wave] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 8; ++w) top = fmaxf(top, lead[w]);
  const float own = pl == 0.f ? 0.f : exp2_ratio(pm, top);
  weights[tid] = own;
  float sum = part_sum(pm, pl, own, top);
#pragma unroll
  for (int k = 32; k > 0; k /= 2) sum += __shfl_xor(sum, k, 64);
  if (lane == 0) total[wave] = sum;
  __syncthreads();
  const int share = tid / (kSplitDims / 4), at = tid % (kSplitDims / 4);
  const int dim = static_cast<int>(blockIdx.z) * kSplitDims + 4 * at;
  v4f o = {0.f, 0.f, 0.f, 0.f};
  for (int i0 = share; i0 < parts; i0 += U * kShares) {
    v4f x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      x[u] = *reinterpret_cast<const v4f*>(
          st.part_o + merge_slot(job, st.part_rows, local, min(i0 + u * kShares, parts - 1)) * L + dim);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * kShares;
      const float f = i < parts ? weights[i] : 0.f;
      if (f != 0.f) o += x[u] * f;
    }
  }
  sums[share][at] = o;
  __syncthreads();
  if (share != 0) return;
  sum = 0.f;
#pragma unroll
  for (int w = 0; w < 8; ++w) sum += total[w];
#pragma unroll
  for (int k = 1; k < kShares; ++k) o += sums[k][at];
  *reinterpret_cast<v4f*>(merge_out(a, job, r) + dim) = o * row_factor(sum, false, 1.0f);
}

// ----------------------------------------------------------------- host ----
// A workgroup a CU: a tile of 32 rows of 576 elements takes 36 KB of LDS.
constexpr std::size_t kGroups = 256;
static_assert(kGroups + 1 <= kMostParts);

// Rows of a unit.  The wavefronts of 16-row units need not wait for each other, but
// each unit brings the pages into LDS for itself.  Two units of the same pages are
// ahead of one of 64 rows (pages cold; one sequence of 131071 tokens, 32 rows, bf16: 52
// us for 61; 64 of 2048, fp32: 136 for 178), and up to 256 units of fp8 pages, whose
// rows are half as long (64 of 2048, 64 rows: 53 for 61; 48 of them, 128 rows: 85 for
// 81); three or four of bf16 or fp32 pages are not (64 rows, bf16: 74 for 66; 64 of
// 2048, 40 rows, fp32: 200 for 179).  With a tile or less for each workgroup the join of
// what a workgroup's wavefronts have takes longer than a tile (one sequence of 500
// tokens, 16 rows: 20 us for 16).
std::size_t unit_rows(const LatentArgs& a) {
  const std::size_t rows = a.q_heads * a.tokens, units = a.batch * ((rows + 15) / 16);
  const std::size_t tile_pages = a.page_type == PageType::kF32 ? 1 : 2;
  const std::size_t tiles = a.batch * ((a.max_blocks + tile_pages - 1) / tile_pages);
  if (tiles <= kGroups) return 64;
  return rows <= 32 || (a.page_type == PageType::kFP8 && units <= kGroups) ? 16 : 64;
}

// Room for units of 64 rows, where there are as many.
struct LatentLayout {
  LatentLayout(std::size_t rows, std::size_t latent) {
    const std::size_t part_rows = rows <= 16 ? 16 : 64;
    auto take = [&](std::size_t n) {
      const std::size_t at = bytes;
      bytes += align256(n);
      return at;
    };
    jobs = take(kGroups * sizeof(LatentJob));
    part_ml = take(2 * kGroups * part_rows * 2 * sizeof(float));
    part_o = take(2 * kGroups * part_rows * latent * sizeof(float));
  }
  std::size_t jobs, part_ml, part_o, bytes = 0;
};

template <int PF, int L>
hipError_t launch_latent(const LatentKernelArgs& k, const LatentStream& st, std::size_t rb,
                         hipStream_t stream) {
  if (rb == 16) {
    latent_kernel<PF, L, false><<<dim3(static_cast<unsigned>(kGroups)), 64 * kWaves, 0, stream>>>(k, st);
  } else {
    latent_kernel<PF, L, true><<<dim3(static_cast<unsigned>(kGroups)), 64 * kWaves, 0, stream>>>(k, st);
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const std::size_t jobs =
      st.by_unit != 0 ? static_cast<std::size_t>(k.batch) * st.row_blocks : kGroups;
  const unsigned rows = static_cast<unsigned>(std::min<std::size_t>(rb, static_cast<std::size_t>(k.rows)));
  if (jobs * kFewParts <= kGroups) {
    latent_split_merge_kernel<L>
        <<<dim3(static_cast<unsigned>(jobs), rows, L / kSplitDims), 512, 0, stream>>>(k, st, static_cast<int>(rb));
  } else {
    latent_merge_kernel<L><<<dim3(static_cast<unsigned>(jobs), (rows + 3) / 4), 256, 0, stream>>>(
        k, st, static_cast<int>(rb));
  }
  return hipGetLastError();
}

template <int PF>
hipError_t launch_page_type(const LatentKernelArgs& k, const LatentStream& st, std::size_t rb,
                            std::size_t latent, hipStream_t stream) {
  return latent == 512 ? launch_latent<PF, 512>(k, st, rb, stream)
                       : launch_latent<PF, 256>(k, st, rb, stream);
}

}  // namespace

std::size_t latent_workspace_bytes(std::size_t, std::size_t q_heads, std::size_t tokens,
                                   std::size_t latent) {
  return LatentLayout(q_heads * tokens, latent).bytes;
}

bool latent_fits(const LatentArgs& a) {
  // Ranges, and places in them, are counted in 32 bits: of 2^38 places, a group's
  // are 2^30 at most.
  const std::size_t rows = a.q_heads * a.tokens;
  const std::size_t units = a.batch * ((rows + 15) / 16);
  return units == 0 || a.max_blocks + 2 + start_cost<false>() <= (std::size_t{1} << 38) / units;
}

hipError_t launch_latent_attention(const LatentArgs& a, hipStream_t stream) {
  if (a.batch == 0 || a.q_heads == 0 || a.tokens == 0) return hipSuccess;
  if (!latent_fits(a)) return hipErrorInvalidValue;
  const LatentLayout layout(a.q_heads * a.tokens, a.latent);
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
  k.rows = static_cast<int>(a.q_heads * a.tokens);
  k.physical_blocks = static_cast<std::uint32_t>(a.physical_blocks);
  k.qscale = kLog2e * a.scale * (a.page_type == PageType::kFP8 ? a.page_scale : 1.0f);
  k.page_scale = a.page_scale;
  auto* const base = static_cast<unsigned char*>(a.workspace);
  LatentStream st{};
  st.jobs = reinterpret_cast<LatentJob*>(base + layout.jobs);
  st.part_ml = reinterpret_cast<float*>(base + layout.part_ml);
  st.part_o = reinterpret_cast<float*>(base + layout.part_o);
  st.groups = static_cast<int>(kGroups);
  const std::size_t rb = unit_rows(a), row_blocks = (a.q_heads * a.tokens + rb - 1) / rb;
  st.part_rows = rb == 16 || a.q_heads * a.tokens <= 16 ? 16 : 64;
  st.row_blocks = static_cast<int>(row_blocks);
  st.share = static_cast<int>(latent_share(kGroups, row_blocks));
  st.by_unit = a.batch * row_blocks <= kGroups ? 1 : 0;
  switch (a.page_type) {
    case PageType::kBF16: return launch_page_type<1>(k, st, rb, a.latent, stream);
    case PageType::kFP8: return launch_page_type<2>(k, st, rb, a.latent, stream);
    default: return launch_page_type<0>(k, st, rb, a.latent, stream);
  }
}

}  // namespace helix::hip
