// Attention of a tree of drafted tokens over paged histories.
//
// Row t of sequence b (node t, in every query head) attends to the sequence's
// whole history and to the tree rows of its ancestors and itself:
//
//   out_t = sum_j p_tj v_j / sum_j p_tj,  p_tj = exp(q_t . k_j / sqrt(128) - m_t),
//
// j over the lengths[b] paged tokens and the nodes on t's way to its root.
// All rows of a (sequence, kv head), its query heads times the nodes, lie one
// behind another in memory and form a unit (of up to RB rows): one pass over
// the unit's keys serves them all.
//
// Work split.  A unit's keys are blocks of 32: its history's, then its tree's.
// A fixed grid of workgroups takes equal ranges of the flat list of all
// units' blocks, whatever the lengths.  A unit inside one range is finished
// there; one that crosses ranges leaves a partial (maximum, sum, output) per
// range, and tree_merge_kernel joins them.  A workgroup leaves at most two
// partials, its first unit's and its last one's, so the workspace depends on
// the grid, not on the batch.
//
// Matrix form.  Per block, scores are S^T = K Q^T and outputs O^T += V^T P^T
// on v_mfma_f32_16x16x32: a lane holds keys of one query row, so a row's
// maximum and sum take two cross-lane steps and its probabilities are an
// operand as they are.  fp32 factors are sums of 16-bit terms, each product
// of terms exact in fp32:
// - bf16 pages: elements are one bf16 term, queries and probabilities three
//   (24 bits): 3 products;
// - fp8 pages: codes are exact in fp16, queries and probabilities two fp16
//   terms (22 bits and a sign: the rounding of an fp32 number): 2 products.
//   Terms must stay above fp16's smallest numbers: a query row is scaled by a
//   power of two that puts its largest element in [2^10, 2^11), and
//   probabilities (with them sums and outputs) carry a factor of 2^8;
// - fp32 pages: three bf16 terms on either side, less the products below
//   2^-26 of the largest: 6 products, 2.7 times the rate of fp32 matrix
//   instructions.
// Elements are split or widened once per workgroup on their way into LDS.
//
// Special values.  Terms of infinities, a 0 times an infinity and values that
// a row does not see can only show as a NaN in the row's sum or outputs.  A
// tile of 16 rows that ends a part with one is marked, and tree_merge_kernel
// computes that part of it again with exact_row.
//
// Measured (both launches, after the first hundred calls, which take up to a fifth
// longer): 64 sequences of 512 to 8192 tokens, 32/8 heads, trees of 16 nodes: fp32
// pages 360 us and bf16 pages 182 us, both at 4.2 TB/s of pages; loads and LDS
// writes alone take 330 and 165, products alone 306 and 150.  Trees of 64 nodes,
// fp8 pages: 454 us (885 TFLOP/s of fp16 products), vector work (16 exponentials
// and as many splits a lane and block) beside the matrix instructions.  One
// sequence of 131071, 33 nodes, bf16: 303 us.
#include "prefill_bmma.hpp"
#include "tree_exact.hpp"

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <type_traits>

namespace helix::hip {
namespace {

using namespace tree_detail;
using prefill_detail::bmma_k_at;
using prefill_detail::bmma_v_at;
using prefill_detail::row_max;
using prefill_detail::row_sum;
using prefill_detail::uniform_read;
using prefill_detail::v4f;
using prefill_detail::v4s;
using prefill_detail::v8bf;
using prefill_detail::v8s;

typedef unsigned v2u __attribute__((ext_vector_type(2)));
typedef unsigned v4u __attribute__((ext_vector_type(4)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef float v2f __attribute__((ext_vector_type(2)));
typedef __bf16 v2bf __attribute__((ext_vector_type(2)));

constexpr int kBlock = 32;  // keys of a block: two pages

// Terms of a page element and of the fp32 factor against it.
constexpr int page_terms(int pf) { return pf == 0 ? 3 : 1; }
constexpr int row_terms(int pf) { return pf == 2 ? 2 : 3; }
// fp8 pages: the factor on probabilities, and its logarithm.
constexpr float kProbScale = 256.0f, kProbLog = 8.0f;
// A row's reference stays while no score is above it by more than this (log2
// units): fp16's largest number is 2^16.
constexpr float kSlack = 7.0f;

constexpr int kMaxTiles = 16;           // 16-row tiles of a unit

// A unit to join: the one that the group's range ends without starting it.
struct TreeJob {
  int b, kvh, rb;  // sequence (-1: none), kv head, row block
  int first;       // group whose range starts the unit,
  int head;        // with so many of its blocks,
  int each;        // and the blocks of a later range
};

struct TreeStream {
  float* part_o;   // [2 * groups, RB, 128]
  float* part_ml;  // [2 * groups, RB, 2]
  TreeJob* jobs;   // [groups]
  // Tiles to compute again: of partials [2 * groups, kMaxTiles], and of
  // finished units [units, kMaxTiles] (0 for units that are joined).
  unsigned char* part_marks;
  unsigned char* unit_marks;
  int groups;
  int row_blocks;  // units of a (sequence, kv head)
};

// x = t[0] + t[1] (+ t[2]), each rounded to nearest; two numbers at a time,
// packed into words.
template <int PF>
__device__ __forceinline__ void split_pair(float x, float y, unsigned (&t)[3]) {
  if constexpr (PF == 2) {
    const v2h hi = __builtin_convertvector((v2f{x, y}), v2h);
    // One mixed-precision instruction a remainder: the compiler must not see
    // that the factor is -1.
    float minus = -1.0f;
    asm("" : "+s"(minus));
    x = __builtin_fmaf(static_cast<float>(hi[0]), minus, x);
    y = __builtin_fmaf(static_cast<float>(hi[1]), minus, y);
    t[0] = __builtin_bit_cast(unsigned, hi);
    t[1] = __builtin_bit_cast(unsigned, __builtin_convertvector((v2f{x, y}), v2h));
  } else {
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      const v2bf h = __builtin_convertvector((v2f{x, y}), v2bf);
      t[i] = __builtin_bit_cast(unsigned, h);
      x -= __uint_as_float(t[i] << 16);
      y -= __uint_as_float(t[i] & 0xffff0000u);
    }
  }
}

// The larger of two numbers, NaN where either is one (one instruction; fmaxf
// takes two more to quiet its arguments).
__device__ __forceinline__ float larger(float a, float b) {
  return __builtin_elementwise_maximum(a, b);
}

template <int PF>
__device__ __forceinline__ v4f matrix_step(v4u a, v4u b, v4f c) {
  if constexpr (PF == 2) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a),
                                                  __builtin_bit_cast(v8h, b), c, 0, 0, 0);
  } else {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a),
                                                   __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
  }
}

// Eight fp8 codes as fp16.
__device__ __forceinline__ v4u codes_fp16(unsigned w0, unsigned w1) {
  return v4u{
      __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w0, 1.0f, false)),
      __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w0, 1.0f, true)),
      __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w1, 1.0f, false)),
      __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w1, 1.0f, true))};
}

// 16 bytes of each plane that 8 elements become in LDS: from 8 fp32 values (a
// tree row, or an fp32 page), rounded onto the page grid.
template <int PF>
__device__ __forceinline__ void chunk_of_rows(v4f x0, v4f x1, float scale,
                                              v4u (&t)[page_terms(PF)]) {
  if constexpr (PF == 0) {
    unsigned w[4][3];
    split_pair<0>(x0[0], x0[1], w[0]);
    split_pair<0>(x0[2], x0[3], w[1]);
    split_pair<0>(x1[0], x1[1], w[2]);
    split_pair<0>(x1[2], x1[3], w[3]);
#pragma unroll
    for (int i = 0; i < 3; ++i) t[i] = v4u{w[0][i], w[1][i], w[2][i], w[3][i]};
  } else if constexpr (PF == 1) {
    t[0] = v4u{bf16_pack(x0[0], x0[1]), bf16_pack(x0[2], x0[3]), bf16_pack(x1[0], x1[1]),
               bf16_pack(x1[2], x1[3])};
  } else {
    t[0] = codes_fp16(fp8_pack4_scaled(make_float4(x0[0], x0[1], x0[2], x0[3]), scale),
                      fp8_pack4_scaled(make_float4(x1[0], x1[1], x1[2], x1[3]), scale));
  }
}

// Whether the two wavefronts of each SIMD take turns (tree_mma_body), and the LDS
// buffers that takes: an item is put there two steps before its use, or one step,
// or (fp32 pages, whose three planes would take the space of a second workgroup)
// just before it.  (131071 bf16 tokens, 33 nodes: 302 us in turns, 322 without.)
constexpr bool in_turns(int pf, int waves, int tiles) {
  return pf == 1 && waves == 8 && tiles == 2;
}
constexpr int stage_buffers(int pf, int waves, int tiles) {
  return pf == 0 ? 1 : in_turns(pf, waves, tiles) ? 3 : 2;
}

// Items on their way from memory to registers.  (64 bf16 sequences of 16 nodes:
// 182 us with two, 183 with one; 32 of them 110 with two, 111 with one.  Three, and
// two of fp32 pages, gained nothing; fp8 pages gained more from the registers of a
// third workgroup on the CU.)
constexpr int load_depth(int pf, int tiles) { return pf == 1 && tiles == 1 ? 2 : 1; }

template <int PF, int W, int RT>
struct TreeShared {
  // Item i: K of block i and V of block i - 1.
  struct Item {
    __align__(1024) unsigned char k[page_terms(PF)][kBlock * 2 * D];
    __align__(1024) unsigned char v[page_terms(PF)][kBlock * 2 * D];
  };
  Item item[stage_buffers(PF, W, RT)];
  // The third terms of the query operands: [tile][step][lane].
  __align__(16) v4u low[row_terms(PF) == 3 ? W * RT : 1][row_terms(PF) == 3 ? 4 : 1][64];
};

// A place in the flat list of blocks.
struct TreeCursor {
  int b, kvh, rb, blk;
  int hist, count, nbh, nb;  // the sequence's tokens, nodes, history blocks, blocks
  int bad;                   // its length lies outside its table
};

__device__ __forceinline__ void load_sequence(const TreeKernelArgs& a, TreeCursor& c) {
  const int hist = uniform_read(a.lengths + c.b);
  c.bad = hist < 0 || hist > a.max_blocks * P;
  c.hist = c.bad ? 0 : hist;
  c.count = a.nodes;
  if (a.node_counts != nullptr) c.count = min(max(uniform_read(a.node_counts + c.b), 0), a.nodes);
  c.nbh = c.count > 0 ? (c.hist + kBlock - 1) / kBlock : 0;
  c.nb = c.nbh + (c.count + kBlock - 1) / kBlock;
}

__device__ __forceinline__ long long uniform_long(long long v) {
  const unsigned lo = __builtin_amdgcn_readfirstlane(static_cast<unsigned>(v));
  const unsigned hi =
      __builtin_amdgcn_readfirstlane(static_cast<unsigned>(static_cast<unsigned long long>(v) >> 32));
  return static_cast<long long>(static_cast<unsigned long long>(hi) << 32 | lo);
}

__device__ __forceinline__ int lane_blocks(const TreeKernelArgs& a, int b) {
  if (b >= a.batch) return 0;
  const int count = clamped_nodes(a, b);
  if (count == 0) return 0;
  return (max(clamped_history(a, b), 0) + kBlock - 1) / kBlock + (count + kBlock - 1) / kBlock;
}

// Inclusive sums over the wavefront.
__device__ __forceinline__ long long lane_scan(long long v, int lane) {
  long long sum = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const long long t = __shfl_up(sum, o, 64);
    if (lane >= o) sum += t;
  }
  return sum;
}

// This group's range of blocks [g0, g1) (ranges of `each`) and its first place.
struct TreeRange {
  long long g0, g1, each;  // (a range's length fits 31 bits: tree_fits)
};
__device__ __forceinline__ TreeRange first_place(const TreeKernelArgs& a, const TreeStream& st,
                                                 int group, int lane, TreeCursor& c) {
  long long per_head = 0;
#pragma unroll 4
  for (int b0 = 0; b0 < a.batch; b0 += 64) per_head += lane_blocks(a, b0 + lane);
  per_head = uniform_long(__shfl(lane_scan(per_head, lane), 63, 64)) * st.row_blocks;
  const long long total = per_head * a.kv_heads;
  TreeRange r{};
  // (Ranges of one block where there are few: 121 tokens and 5 nodes take 14 us
  // in both launches, 20 with ranges of four.)
  r.each = uniform_long(max((total + st.groups - 1) / st.groups, 1ll));
  r.g0 = uniform_long(group * r.each);
  r.g1 = uniform_long(min(r.g0 + r.each, total));
  if (r.g0 >= r.g1) return r;
  c.kvh = __builtin_amdgcn_readfirstlane(static_cast<int>(r.g0 / per_head));
  const long long rem = r.g0 - c.kvh * per_head;
  long long base = 0;
  int nb = lane_blocks(a, lane);
  for (int b0 = 0; b0 < a.batch; b0 += 64) {
    const int next = lane_blocks(a, b0 + 64 + lane);
    const long long sum = lane_scan(nb, lane);
    const long long from = (base + sum - nb) * st.row_blocks, to = (base + sum) * st.row_blocks;
    const unsigned long long hit = __ballot(from <= rem && rem < to);
    if (hit != 0) {
      const int src = __ffsll(static_cast<long long>(hit)) - 1;
      c.b = __builtin_amdgcn_readfirstlane(b0 + src);
      load_sequence(a, c);
      const int in = static_cast<int>(rem - uniform_long(__shfl(from, src, 64)));
      c.rb = __builtin_amdgcn_readfirstlane(in / c.nb);
      c.blk = __builtin_amdgcn_readfirstlane(in - c.rb * c.nb);
      break;
    }
    base += uniform_long(__shfl(sum, 63, 64));
    nb = next;
  }
  return r;
}

// The next place; only called where there is one.
__device__ __forceinline__ void advance(const TreeKernelArgs& a, const TreeStream& st,
                                        TreeCursor& c) {
  if (++c.blk < c.nb) return;
  c.blk = 0;
  if (++c.rb < st.row_blocks) return;
  c.rb = 0;
  do {
    if (++c.b == a.batch) {
      c.b = 0;
      ++c.kvh;
    }
    load_sequence(a, c);
  } while (c.nb == 0);
}

// The rows of a block that is, or is not, one of tree rows.
struct TreeSource {
  std::size_t at;  // element offset of its tree rows
  int tree;        // tree rows
  int rows;        // rows of it that are the sequence's
  int bad;         // of a sequence with a length or page that is none
};

// W wavefronts of RT tiles of 16 query rows: units of RB = 16 W RT rows.
//
// Step n of a wavefront: it puts its share of a later item (K of a block, V of
// the block before) from registers into LDS and sends for the next one's; turns
// block n's scores into probabilities; and, past a barrier, takes block n's P V
// and the scores of block n + 1, matrix instructions one behind another.
// Where they take turns, the first four wavefronts and the others are half a step
// apart, with a second barrier: one of a SIMD's two is at its matrix instructions
// while the other is at its vector instructions.
// Steps whose items are whole pages of one unit run in a loop of their own, where
// the compiler knows which loads are on their way.
template <int PF, int W, int RT>
__device__ __forceinline__ void tree_mma_body(const TreeKernelArgs& a, const TreeStream& st,
                                              TreeShared<PF, W, RT>& sh) {
  // Four tree rows are a job of a wavefront: eight for K, and the same rows' for
  // V.  Of pages a job is what loads of 16 bytes a lane bring, without gaps: four
  // rows in two loads or one, or eight rows of fp8.
  static_assert(8 % W == 0);
  constexpr int NT = 8 / W;
  constexpr int kJobRows = PF == 2 ? 8 : 4;
  constexpr int NJ = kBlock / kJobRows / W;
  constexpr int RW = PF == 0 ? 2 : 1;
  constexpr int RB = 16 * W * RT;
  constexpr int KT = page_terms(PF), QT = row_terms(PF);
  constexpr int NB = stage_buffers(PF, W, RT);
  constexpr bool kTurns = in_turns(PF, W, RT);
  constexpr int DEPTH = load_depth(PF, RT);
  // Blocks from the one whose scores are taken to the one located last.
  constexpr int kLead = kTurns ? DEPTH + 1 : DEPTH;
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, grp = lane >> 4;
  const int group = static_cast<int>(blockIdx.x);
  // (Between scheduling barriers: register work that the compiler moves across
  // lands among the matrix instructions behind it.)
  auto barrier = [] {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };

  if (tid == 0) st.jobs[group] = TreeJob{-1, 0, 0, 0, 0, 0};
  TreeCursor cur{};
  const TreeRange range = first_place(a, st, group, lane, cur);
  if (range.g0 >= range.g1) return;
  const int blocks = static_cast<int>(range.g1 - range.g0);

  // Pages of the (sequence, kv head) being loaded, 64 at a time: lane i holds
  // the byte offset of page pages_at + i in the pools.  (Behind the history the
  // last page is read again; a page outside the pool is not read.)
  constexpr int kElem = PF == 0 ? 4 : PF == 1 ? 2 : 1;
  unsigned page_lo = 0, page_hi = 0;
  int pages_of = -1, pages_at = 0;
  int bad_page = 0;  // some of them are none
  // key_at[i]: K of job i in the page pool, 16 bytes a lane from there on, of the
  // block located last; V is as far on in its pool, one block later.
  // Before any block of pages: page 0.
  unsigned long long key_at[NJ], value_at[NJ];
#pragma unroll
  for (int i = 0; i < NJ; ++i) {
    key_at[i] = reinterpret_cast<std::uintptr_t>(a.key_pool);
    value_at[i] = reinterpret_cast<std::uintptr_t>(a.value_pool);
  }
  const unsigned long long value_off = static_cast<unsigned long long>(
      static_cast<const unsigned char*>(a.value_pool) - static_cast<const unsigned char*>(a.key_pool));
  auto job = [&](int i) { return wave + W * i; };
  auto job_row = [&](int i) { return kJobRows * job(i); };
  auto locate_pages = [&](int first) {
#pragma unroll
    for (int i = 0; i < NJ; ++i) {
      const int n = first + job_row(i) / P;
      const unsigned lo = __builtin_amdgcn_readlane(page_lo, n);
      const unsigned hi = __builtin_amdgcn_readlane(page_hi, n);
      key_at[i] = (static_cast<unsigned long long>(hi) << 32 | lo) +
                  static_cast<unsigned>(job_row(i) % P * (D * kElem)) +
                  reinterpret_cast<std::uintptr_t>(a.key_pool);
    }
  };
  auto locate = [&](const TreeCursor& c) {
    TreeSource s{};
    s.bad = c.bad;
    if (__builtin_expect(c.blk >= c.nbh, 0)) {
      const int first = (c.blk - c.nbh) * kBlock;
      s.tree = 1;
      s.rows = c.count - first;
      s.at = ((static_cast<std::size_t>(c.b) * a.kv_heads + c.kvh) * a.nodes + first) * D;
      return s;
    }
    s.rows = c.hist - c.blk * kBlock;
    const int unit = c.kvh * a.batch + c.b;
    int first = 2 * c.blk - pages_at;
    if (__builtin_expect(pages_of != unit || first < 0 || first >= 64, 0)) {
      pages_of = unit;
      pages_at = 2 * c.blk;
      first = 0;
      unsigned page = a.tables[static_cast<std::size_t>(c.b) * a.max_blocks +
                               min(pages_at + lane, (c.hist - 1) / P)];
      const bool outside = page >= a.physical_blocks;
      bad_page = __ballot(outside) != 0 ? 1 : 0;
      if (outside) page = 0;
      const unsigned long long at =
          (static_cast<unsigned long long>(page) * a.kv_heads + c.kvh) * (P * D * kElem);
      page_lo = static_cast<unsigned>(at);
      page_hi = static_cast<unsigned>(at >> 32);
    }
    s.bad |= bad_page;
    locate_pages(first);
    return s;
  };

  using Raw = std::conditional_t<PF == 0, v4f, v4u>;
  using Global = const __attribute__((address_space(1))) Raw*;
  using GlobalBytes = const __attribute__((address_space(1))) unsigned char*;
  const unsigned lane_at = static_cast<unsigned>(lane) * 16u;
  // (A unit reads each byte once.  Where its head's rows are several units, past
  // 256 rows, or 128 with fp8 pages, each of them reads the pages.)
  auto stream = [&](unsigned long long at, int w) {
    return __builtin_nontemporal_load(
        reinterpret_cast<Global>(reinterpret_cast<GlobalBytes>(at + 1024u * w) + lane_at));
  };
  using GlobalRows = const __attribute__((address_space(1))) v4f*;
  Raw key_raw[DEPTH][NJ * RW], value_raw[DEPTH][NJ * RW];
  auto load_pages = [&](auto set) {
    constexpr int S = decltype(set)::value;
    // (Or loads from an address that was loaded from before become copies.)
    asm volatile("" ::: "memory");
#pragma unroll
    for (int i = 0; i < NJ; ++i) {
#pragma unroll
      for (int w = 0; w < RW; ++w) {
        key_raw[S][RW * i + w] = stream(key_at[i], w);
      }
    }
#pragma unroll
    for (int i = 0; i < NJ; ++i) {
#pragma unroll
      for (int w = 0; w < RW; ++w) {
        value_raw[S][RW * i + w] = stream(value_at[i], w);
      }
    }
  };
  // A job's loads into the planes `to`, chunks of 8 elements at at(row, chunk);
  // rows from `rows` on become 0.
  auto put_raw = [&](unsigned char* to, auto at, int row0, const Raw* x, int rows) {
    constexpr std::size_t kPlane = kBlock * 2 * D;
    if constexpr (PF == 0) {
#pragma unroll
      for (int w = 0; w < RW; ++w) {
        const int row = row0 + 2 * w + (lane >> 5);
        unsigned p[2][3];
        split_pair<0>(x[w][0], x[w][1], p[0]);
        split_pair<0>(x[w][2], x[w][3], p[1]);
#pragma unroll
        for (int n = 0; n < KT; ++n) {
          *reinterpret_cast<v2u*>(to + n * kPlane + at(row, (lane & 31) >> 1) + 8 * (lane & 1)) =
              row >= rows ? v2u{0u, 0u} : v2u{p[0][n], p[1][n]};
        }
      }
    } else if constexpr (PF == 1) {
      const int row = row0 + grp;
      *reinterpret_cast<v4u*>(to + at(row, col)) = row >= rows ? v4u{0u, 0u, 0u, 0u} : x[0];
    } else {
      const int row = row0 + (lane >> 3);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        *reinterpret_cast<v4u*>(to + at(row, 2 * (lane & 7) + h)) =
            row >= rows ? v4u{0u, 0u, 0u, 0u} : codes_fp16(x[0][2 * h], x[0][2 * h + 1]);
      }
    }
  };
  auto k_place = [](int row, int chunk) { return bmma_k_at(row, chunk); };
  auto v_place = [](int row, int chunk) { return bmma_v_at(row, chunk); };
  auto put_key_raw = [&](auto set, int buf, int i) {
    put_raw(sh.item[buf].k[0], k_place, job_row(i), key_raw[decltype(set)::value] + RW * i, kBlock);
  };
  auto put_value_raw = [&](auto set, int buf, int i, int rows) {
    put_raw(sh.item[buf].v[0], v_place, job_row(i), value_raw[decltype(set)::value] + RW * i, rows);
  };
  // An item of whole pages into LDS.
  auto store_pages = [&](auto set, int buf) {
#pragma unroll
    for (int i = 0; i < NJ; ++i) {
      put_key_raw(set, buf, i);
      put_value_raw(set, buf, i, kBlock);
    }
  };
  // Any item: what was loaded, or (`s.tree`) rows read now.  (Those read ahead
  // into the pages' registers would have the pages' loads waited for at once.)
  auto from_rows = [&](const TreeSource& s, const float* rows, float scale, int i,
                       v4u (&t)[KT]) {
    const auto x = reinterpret_cast<GlobalRows>(reinterpret_cast<std::uintptr_t>(
        rows + s.at + min(4 * job(i) + grp, s.rows - 1) * D + col * 8));
    chunk_of_rows<PF>(x[0], x[1], scale, t);
  };
  auto store_key = [&](auto set, int buf, const TreeSource& s) {
    if (s.tree == 0) {
#pragma unroll
      for (int i = 0; i < NJ; ++i) put_key_raw(set, buf, i);
      return;
    }
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      v4u t[KT];
      from_rows(s, a.tree_key, a.k_scale, i, t);
#pragma unroll
      for (int n = 0; n < KT; ++n) {
        *reinterpret_cast<v4u*>(sh.item[buf].k[n] + bmma_k_at(4 * job(i) + grp, col)) = t[n];
      }
    }
  };
  // (Rows behind the sequence's must be finite.)
  auto store_value = [&](auto set, int buf, const TreeSource& s) {
    if (s.tree == 0) {
#pragma unroll
      for (int i = 0; i < NJ; ++i) put_value_raw(set, buf, i, s.rows);
      return;
    }
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      v4u t[KT];
      from_rows(s, a.tree_value, a.v_scale, i, t);
#pragma unroll
      for (int n = 0; n < KT; ++n) {
        *reinterpret_cast<v4u*>(sh.item[buf].v[n] + bmma_v_at(4 * job(i) + grp, col)) =
            4 * job(i) + grp >= s.rows ? v4u{0u, 0u, 0u, 0u} : t[n];
      }
    }
  };

  // The wavefront's rows of the unit: tile t's row `col`, from tile_row(t) on.
  auto tile_row = [&](int t) { return (t * W + wave) * 16; };
  bool live = false;  // the first of them has rows
  v4u qop[RT][2][4];  // (the third term of three is in LDS)
  float unscale[RT];  // fp8 pages: what undoes the row's power of two
  int parent = -1;    // of node `lane`
  v4f o[RT][8];       // o[t][dt][i]: dim 16 dt + 4 grp + i of row col
  float m[RT], l[RT];
  bool finite = false;  // every row's reference is a number
  unsigned long long broken = 0;  // the nodes with a wrong parent on their way
  auto unit_rows = [&](const TreeCursor& c) {
    return (static_cast<std::size_t>(c.b) * a.q_heads +
            static_cast<std::size_t>(c.kvh) * (a.q_heads / a.kv_heads)) *
           a.nodes;
  };
  auto start = [&](const TreeCursor& c) {
    const float scale = PF == 2 ? a.qscale * a.k_scale : a.qscale;
    parent = node_parent(a, c.b, c.count, lane);
    live = c.rb * RB + tile_row(0) < a.rows;
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      const int row = c.rb * RB + tile_row(t) + col;
      v4f x[4][2];
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        x[s][0] = x[s][1] = v4f{0.f, 0.f, 0.f, 0.f};
        if (row < a.rows) {
          const auto* q =
              reinterpret_cast<const v4f*>(a.query + (unit_rows(c) + row) * D + 32 * s + 8 * grp);
          x[s][0] = q[0];
          x[s][1] = q[1];
        }
      }
      float grow = scale;
      if constexpr (PF == 2) {
        float most = 0.f;
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            most = fmaxf(most, fmaxf(fmaxf(fabsf(x[s][w][0]), fabsf(x[s][w][1])),
                                     fmaxf(fabsf(x[s][w][2]), fabsf(x[s][w][3]))));
          }
        most = row_max(most);
        // most * 2^(10 - e) in [2^10, 2^11), as far as 2^(10 - e) is a normal
        // number.
        const int e = min(max(static_cast<int>(__float_as_uint(most) >> 23) - 127, -110), 120);
        grow = __uint_as_float(static_cast<unsigned>(127 + 10 - e) << 23);
        unscale[t] = __uint_as_float(static_cast<unsigned>(127 - 10 + e) << 23) * scale;
      }
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        unsigned w[4][3];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          split_pair<PF>(x[s][i >> 1][2 * (i & 1)] * grow, x[s][i >> 1][2 * (i & 1) + 1] * grow, w[i]);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) qop[t][i][s] = v4u{w[0][i], w[1][i], w[2][i], w[3][i]};
        if constexpr (QT == 3) {
          sh.low[wave * RT + t][s][lane] = v4u{w[0][2], w[1][2], w[2][2], w[3][2]};
        }
      }
#pragma unroll
      for (int dt = 0; dt < 8; ++dt) o[t][dt] = v4f{0.f, 0.f, 0.f, 0.f};
      m[t] = -INFINITY;
      l[t] = 0.f;
    }
    broken = 0;
    finite = false;
  };

  // Scores of a block: sc[t][h][i] is key 16 h + 4 grp + i of tile t's row col.
  const unsigned k_at = bmma_k_at(col, grp);
  // (Operands come out of LDS ahead of the instructions that take them: a half
  // block's 32 dims, or a tile's 16, are 48 to 96 cycles of these.)
  constexpr int kAhead = PF == 0 || RT == 1 ? 2 : PF == 2 ? 3 : 4;
  auto scores = [&](auto tiles, int buf, v4f (&sc)[RT][2]) {
    constexpr int LT = decltype(tiles)::value;
    static_assert(QT != 3 || kAhead == 2 || kAhead == 4);
    v4u kop[kAhead][KT], low[2][RT];
    auto read = [&](int u) {  // 32 dims, from 32 (u / 2) on, of keys 16 (u % 2) and on
      const int s = u / 2, h = u % 2;
      // (Of `low` two 32 dims' are there: the next ones' come after the last use.)
      if (QT == 3 && h == (kAhead == 4 ? 1 : 0)) {
#pragma unroll
        for (int t = 0; t < LT; ++t) low[s % 2][t] = sh.low[wave * RT + t][QT == 3 ? s : 0][lane];
      }
#pragma unroll
      for (int i = 0; i < KT; ++i) {
        kop[u % kAhead][i] =
            *reinterpret_cast<const v4u*>(sh.item[buf].k[i] + h * (P * 2 * D) + (k_at ^ (64u * s)));
      }
    };
#pragma unroll
    for (int u = 0; u < kAhead; ++u) read(u);
#pragma unroll
    for (int t = 0; t < LT; ++t) sc[t][0] = sc[t][1] = v4f{0.f, 0.f, 0.f, 0.f};
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int s = u / 2, h = u % 2;
      // Smallest products first.
#pragma unroll
      for (int sum = QT - 1; sum >= 0; --sum) {
#pragma unroll
        for (int i = KT - 1; i >= 0; --i) {
          if (sum - i < 0 || sum - i >= QT) continue;
#pragma unroll
          for (int t = 0; t < LT; ++t) {
            sc[t][h] = matrix_step<PF>(kop[u % kAhead][i],
                                       sum - i == 2 ? low[s % 2][t] : qop[t][sum - i & 1][s],
                                       sc[t][h]);
          }
        }
      }
      if (u + kAhead < 8) read(u + kAhead);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // m[t] is a reference near the row's maximum: it moves where a score is above
  // it by more than kSlack, and what was summed with it.  `vis[t]`: the lane's
  // keys (bit 4 h + i) that the row sees.  Returns whether every key is seen and
  // every reference finite.
  auto maxima = [&](auto tiles, auto whole, const TreeCursor& c, v4f (&sc)[RT][2],
                    unsigned (&vis)[RT]) {
    constexpr int LT = decltype(tiles)::value;
    const bool in_tree = c.blk >= c.nbh;
    const int seen = c.hist - c.blk * kBlock;
    const bool full = decltype(whole)::value || (!in_tree && seen >= kBlock);
#pragma unroll
    for (int t = 0; t < LT; ++t) vis[t] = 0xffu;
    if (__builtin_expect(!full, 0)) {
      unsigned bits[RT];  // the block's keys that the row sees
      if (in_tree) {
        TreeSequence tree{};
        tree_words(parent, c.count, lane, tree);
        broken = __ballot(tree.broken != 0);
#pragma unroll
        for (int t = 0; t < LT; ++t) {
          const int row = c.rb * RB + tile_row(t) + col;
          const unsigned long long w = shfl64(tree.seen, row % a.nodes);
          bits[t] = row < a.rows ? static_cast<unsigned>(w >> ((c.blk - c.nbh) * kBlock)) : 0u;
        }
      } else {
#pragma unroll
        for (int t = 0; t < LT; ++t) bits[t] = (1u << seen) - 1u;
      }
#pragma unroll
      for (int t = 0; t < LT; ++t) {
        vis[t] = ((bits[t] >> (4 * grp)) & 0xfu) | ((bits[t] >> (16 + 4 * grp)) & 0xfu) << 4;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (((vis[t] >> j) & 1u) == 0) sc[t][j >> 2][j & 3] = -INFINITY;
        }
      }
    }
    float mx[RT];
    bool above = false;
#pragma unroll
    for (int t = 0; t < LT; ++t) {
      const v4f x0 = sc[t][0], x1 = sc[t][1];
      mx[t] = larger(larger(larger(x0[0], x0[1]), larger(x0[2], x0[3])),
                     larger(larger(x1[0], x1[1]), larger(x1[2], x1[3])));
      if constexpr (PF == 2) mx[t] *= unscale[t];
      above = above || mx[t] > m[t] + kSlack;
    }
    if (__ballot(above) != 0) {
      finite = true;
#pragma unroll
      for (int t = 0; t < LT; ++t) {
        const float mn = fmaxf(m[t], row_max(mx[t]));
        const float alpha = exp2_ratio(m[t], mn);
#pragma unroll
        for (int dt = 0; dt < 8; ++dt) o[t][dt] *= alpha;
        l[t] *= alpha;
        m[t] = mn;
        finite = finite && __ballot(!(fabsf(mn) < INFINITY)) == 0;
      }
    }
    return full && finite;
  };
  // Probabilities of the block's scores as operands; FINE: maxima() said so.
  auto probabilities = [&](auto tiles, auto fine_tag, v4f (&sc)[RT][2], const unsigned (&vis)[RT],
                           v4u (&pop)[RT][QT]) {
    constexpr int LT = decltype(tiles)::value;
    constexpr bool FINE = decltype(fine_tag)::value;
#pragma unroll
    for (int t = 0; t < LT; ++t) {
      float p[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float x = sc[t][j >> 2][j & 3];
        if constexpr (FINE && PF == 2) {
          p[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(x, unscale[t], kProbLog - m[t]));
        } else if constexpr (FINE) {
          p[j] = __builtin_amdgcn_exp2f(x - m[t]);
        } else if constexpr (PF == 2) {
          p[j] = ((vis[t] >> j) & 1u) != 0 ? exp2_ratio(x * unscale[t], m[t]) * kProbScale : 0.f;
        } else {
          p[j] = ((vis[t] >> j) & 1u) != 0 ? exp2_ratio(x, m[t]) : 0.f;
        }
      }
      // The lane's own keys; the row's four lanes are added at the end.
      l[t] += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
      unsigned w[4][3];
#pragma unroll
      for (int i = 0; i < 4; ++i) split_pair<PF>(p[2 * i], p[2 * i + 1], w[i]);
#pragma unroll
      for (int i = 0; i < QT; ++i) pop[t][i] = v4u{w[0][i], w[1][i], w[2][i], w[3][i]};
    }
  };
  const unsigned v_at =
      bmma_v_at(4 * grp + (col >> 2), 0) + static_cast<unsigned>((col & 3) * 8);
  auto add_values = [&](auto tiles, int buf, const v4u (&pop)[RT][QT]) {
    constexpr int LT = decltype(tiles)::value;
    using LdsV4s = __attribute__((address_space(3))) v4s;
    v4u vop[kAhead][KT];
    auto read = [&](int dt) {
#pragma unroll
      for (int i = 0; i < KT; ++i) {
        unsigned char* const vp = sh.item[buf].v[i] + (v_at ^ (32u * dt));
        const v4s v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsV4s*)(vp));
        const v4s v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsV4s*)(vp + P * 2 * D));
        vop[dt % kAhead][i] =
            __builtin_bit_cast(v4u, __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7));
      }
    };
#pragma unroll
    for (int dt = 0; dt < kAhead; ++dt) read(dt);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int dt = 0; dt < 8; ++dt) {
#pragma unroll
      for (int sum = QT - 1; sum >= 0; --sum) {
#pragma unroll
        for (int i = KT - 1; i >= 0; --i) {
          if (sum - i < 0 || sum - i >= QT) continue;
#pragma unroll
          for (int t = 0; t < LT; ++t) {
            o[t][dt] = matrix_step<PF>(vop[dt % kAhead][i], pop[t][sum - i], o[t][dt]);
          }
        }
      }
      if (dt + kAhead < 8) read(dt + kAhead);
      // (Or the compiler reads each operand where it is needed, and waits.)
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  // Ends the unit's part [from, c.blk] in this range.
  auto finish = [&](const TreeCursor& c, int from, long long g, bool bad) {
    const bool starts = from == 0, ends = c.blk + 1 == c.nb;
    const bool complete = starts && ends;
    const float vscale = PF == 2 ? a.v_scale : 1.0f;
    const int slot = 2 * group + (starts ? 1 : 0);
    const int row_base = complete ? 0 : c.rb * RB;
    float* const rows =
        complete ? a.out + unit_rows(c) * D : st.part_o + static_cast<std::size_t>(slot) * RB * D;
    float* const ml = st.part_ml + static_cast<std::size_t>(slot) * RB * 2;
    const std::size_t unit =
        (static_cast<std::size_t>(c.kvh) * a.batch + c.b) * st.row_blocks + c.rb;
    unsigned char* const marks =
        complete ? st.unit_marks + unit * kMaxTiles : st.part_marks + slot * kMaxTiles;
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      const int row = c.rb * RB + tile_row(t) + col, node = row % a.nodes;
      const bool live = row < a.rows && node < c.count;
      const bool lost = bad || ((broken >> node) & 1) != 0;
      const float sum = row_sum(l[t]);
      bool nan = !(sum < INFINITY);
#pragma unroll
      for (int dt = 0; dt < 8; ++dt)
#pragma unroll
        for (int i = 0; i < 4; ++i) nan = nan || isnan(o[t][dt][i]);
      const bool again = __ballot(nan && live && !lost) != 0;
      if (lane == 0) {
        marks[t * W + wave] = again ? 1 : 0;
        if (ends && !starts) st.unit_marks[unit * kMaxTiles + t * W + wave] = 0;
      }
      if (!live) continue;
      float f = vscale;
      if (complete) f = lost || m[t] == -INFINITY ? NAN : vscale / sum;
      float* const dst = rows + static_cast<std::size_t>(row - row_base) * D + 4 * grp;
#pragma unroll
      for (int dt = 0; dt < 8; ++dt) {
        *reinterpret_cast<float4*>(dst + 16 * dt) =
            make_float4(o[t][dt][0] * f, o[t][dt][1] * f, o[t][dt][2] * f, o[t][dt][3] * f);
      }
      if (!complete && grp == 0) {
        ml[(row - row_base) * 2] = m[t];
        ml[(row - row_base) * 2 + 1] = lost ? NAN : sum;
      }
    }
    if (ends && !starts && tid == 0) {
      const long long start = g - c.blk, first = start / range.each;
      st.jobs[group] = TreeJob{c.b, c.kvh, c.rb, static_cast<int>(first),
                               static_cast<int>((first + 1) * range.each - start),
                               static_cast<int>(range.each)};
    }
  };

  // Item i of the range, K of its block i and V of block i - 1, is put into
  // buffer i % NB from register set i % DEPTH; DEPTH items are on their way.
  // Behind the range, items go on that no one reads.
  using Even = std::integral_constant<int, 0>;
  using Odd = std::integral_constant<int, DEPTH - 1>;
  TreeCursor ahead = cur;        // the block located last,
  int located = 0;               // and its item
  TreeSource key[DEPTH], value;  // of the item to put, and later ones; of the one before
  key[0] = locate(ahead);
  value = key[0];
  unsigned bads = key[0].bad;  // bit i % 32: of block i, as far as it was located
  int item = 0;                // the one to put,
  int into = 0;                // the buffer it goes to
  // Steps from the next one on whose item to put is whole pages, of the unit of
  // the blocks before it, and that locate such a block with page offsets in hand.
  int plain = 0;
  auto locate_next = [&] {
    TreeSource s = key[DEPTH - 1];
    plain = 0;
    if (++located < blocks) {
      advance(a, st, ahead);
      s = locate(ahead);
      bads |= static_cast<unsigned>(s.bad) << (located & 31);
      if (s.tree == 0 && ahead.blk >= kLead && located > kLead) {
        plain = min(min(ahead.nbh - 1, (pages_at >> 1) + 31) - ahead.blk, blocks - 1 - located);
      }
    }
    return s;
  };
  // The item sent for first goes to LDS, and the next one is sent for: of whole
  // pages, or any.
  auto put_pages = [&](auto set) {
    // What was sent for first is there.  (Said here, or the compiler waits for all
    // where the registers are loaded next.)
    __builtin_amdgcn_s_waitcnt(0x0f70 + (DEPTH - 1) * 2 * NJ * RW);
    store_pages(set, into);
    into = into + 1 == NB ? 0 : into + 1;
#pragma unroll
    for (int i = 0; i < NJ; ++i) value_at[i] = key_at[i] + value_off;
    ++ahead.blk;
    locate_pages(2 * ahead.blk - pages_at);
    load_pages(set);
  };
  auto put = [&](auto set) {
    if (item < blocks) store_key(set, into, key[0]);
    if (item > 0 && item <= blocks) store_value(set, into, value);
    into = into + 1 == NB ? 0 : into + 1;
    ++item;
#pragma unroll
    for (int i = 0; i < NJ; ++i) value_at[i] = key_at[i] + value_off;
    value = key[0];
    if constexpr (DEPTH == 2) key[0] = key[1];
    key[DEPTH - 1] = locate_next();
    // (On every path, where what is located is needed or not: loads on some paths
    // only are copied, and so waited for, where the paths meet.)
    load_pages(set);
  };
  load_pages(Even{});
  if constexpr (DEPTH == 2) {
#pragma unroll
    for (int i = 0; i < NJ; ++i) value_at[i] = key_at[i] + value_off;
    key[1] = key[0];
    key[1] = locate_next();
    load_pages(Odd{});
  }
  put(Even{});
  if constexpr (kTurns) put(Odd{});
  start(cur);
  v4f sc[RT][2];
  barrier();
  using All = std::integral_constant<int, RT>;
  scores(All{}, 0, sc);
  const bool second = kTurns && wave >= 4;
  if (second) barrier();
  int from = cur.blk;  // the unit's first block in this range
  int bad = 0;         // of the unit
  int n = 0, buf = 0;
  // Block n's probabilities; item n + 1 goes to LDS meanwhile.
  auto soften = [&](auto tiles, auto whole, v4u (&pop)[RT][QT]) {
    unsigned vis[RT];
    if constexpr (decltype(tiles)::value > 0) {
      if (maxima(tiles, whole, cur, sc, vis)) {
        probabilities(tiles, std::true_type{}, sc, vis, pop);
      } else {
        probabilities(tiles, std::false_type{}, sc, vis, pop);
      }
    }
    barrier();
    buf = buf + 1 == NB ? 0 : buf + 1;
  };
  auto page_step = [&](auto tiles, auto set) {
    if constexpr (NB == 1) barrier();  // the last step's reads are done
    put_pages(set);
    __builtin_amdgcn_sched_barrier(0);
    v4u pop[RT][QT];
    soften(tiles, std::true_type{}, pop);
    if constexpr (decltype(tiles)::value > 0) {
      __builtin_amdgcn_s_setprio(1);
      add_values(tiles, buf, pop);
      scores(tiles, buf, sc);
      __builtin_amdgcn_s_setprio(0);
    }
    if constexpr (kTurns) barrier();
  };
  auto page_steps = [&](auto tiles, int steps) {
#pragma unroll 1
    for (int i = 0; i < steps; i += DEPTH) {
      page_step(tiles, Odd{});
      if constexpr (DEPTH == 2) page_step(tiles, Even{});
    }
  };
  auto step = [&](auto set) {
    if constexpr (NB == 1) barrier();
    put(set);
    __builtin_amdgcn_sched_barrier(0);
    bad |= static_cast<int>(bads >> (n & 31)) & 1;
    bads &= ~(1u << (n & 31));
    v4u pop[RT][QT];
    soften(All{}, std::false_type{}, pop);
    add_values(All{}, buf, pop);
    const bool last = n + 1 == blocks;
    if (last || cur.blk + 1 == cur.nb) {
      finish(cur, from, range.g0 + n, bad != 0);
      if (last) return false;
      advance(a, st, cur);
      from = bad = 0;
      start(cur);
    } else {
      ++cur.blk;
    }
    scores(All{}, buf, sc);
    if constexpr (kTurns) barrier();
    ++n;
    return true;
  };
  // (Step n puts item n + 1, or in turns n + 2.)
  static_assert(!kTurns || DEPTH == 1);
  for (;;) {
    if (plain >= DEPTH) {
      // (Every block on its way is of this unit.)
      bad |= bads != 0 ? 1 : 0;
      bads = 0;
      const int steps = plain / DEPTH * DEPTH;
      // (Or the compiler, not knowing what is on its way from here, waits for all
      // in every second step.)
      if constexpr (DEPTH == 2) __builtin_amdgcn_s_waitcnt(0x0f70);
      // (A tile without rows keeps the scores it had; nothing of it is used.)
      if (RT > 1 || live) {
        page_steps(All{}, steps);
      } else {
        page_steps(std::integral_constant<int, 0>{}, steps);
      }
      plain -= steps;
      n += steps;
      item += steps;
      located += steps;
      cur.blk += steps;
      key[DEPTH - 1].rows -= steps * kBlock;
      if constexpr (DEPTH == 2) key[0].rows = key[1].rows + kBlock;
      value.rows = key[0].rows + kBlock;
    }
    if (!step(Odd{})) break;
    if constexpr (DEPTH == 2) {
      if (!step(Even{})) break;
    }
  }
  if (kTurns && !second) barrier();
}

template <int PF, int W, int RT>
__global__ __launch_bounds__(64 * W)
    __attribute__((amdgpu_waves_per_eu(PF == 2 && RT == 1 ? 3 : 2)))
    void tree_mma_kernel(TreeKernelArgs a, TreeStream st) {
  __shared__ TreeShared<PF, W, RT> sh;
  tree_mma_body<PF, W, RT>(a, st, sh);
}

// Joins the partials of the units that cross ranges: blockIdx.x is the group
// whose range ends such a unit, its partials the first group's second slot and
// the later groups' first ones.  16 lanes take a row, 8 dims each, and 16
// partials' statistics at a time.  (A wavefront a row: 60 us where this takes
// 30, 64 sequences of 64 nodes.)  Marked parts are computed again here; those
// of finished units by the workgroups with blockIdx.y = 0.
constexpr int kMergeRows = 16;
template <int PF>
__global__ __launch_bounds__(256) void tree_merge_kernel(TreeKernelArgs a, TreeStream st,
                                                         int rb_rows) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  auto out_row = [&](int b, int kvh, int row) {
    return a.out + ((static_cast<std::size_t>(b) * a.q_heads +
                     static_cast<std::size_t>(kvh) * (a.q_heads / a.kv_heads)) * a.nodes +
                    row) * D;
  };
  if (blockIdx.y == 0) {
    const std::size_t units = static_cast<std::size_t>(a.batch) * a.kv_heads * st.row_blocks;
    for (std::size_t u = blockIdx.x; u < units; u += gridDim.x) {
      const uint4 marks = *reinterpret_cast<const uint4*>(st.unit_marks + u * kMaxTiles);
      if ((marks.x | marks.y | marks.z | marks.w) == 0) continue;
      const int rb = static_cast<int>(u % st.row_blocks);
      const int b = static_cast<int>(u / st.row_blocks % a.batch);
      const int kvh = static_cast<int>(u / st.row_blocks / a.batch);
      const TreeSequence s = tree_sequence(a, b, lane);
      if (s.count == 0) continue;  // no one wrote its marks
      for (int i = wave; i < rb_rows; i += 4) {
        const int row = rb * rb_rows + i, node = row % a.nodes;
        if (st.unit_marks[u * kMaxTiles + i / 16] == 0 || row >= a.rows || node >= s.count) continue;
        if (((__ballot(s.broken != 0) >> node) & 1) != 0) continue;
        float2 o;
        float m, l;
        exact_row<PF>(a, b, kvh, row, 0, s.hist, 0, s.count, shfl64(s.seen, node), lane, o, m, l);
        const float f = m == -INFINITY ? NAN : 1.0f / l;
        reinterpret_cast<float2*>(out_row(b, kvh, row))[lane] = make_float2(o.x * f, o.y * f);
      }
    }
  }
  const TreeJob job = st.jobs[blockIdx.x];
  if (job.b < 0) return;
  const int part = lane & 15;
  const int local = static_cast<int>(blockIdx.y) * kMergeRows + wave * 4 + (lane >> 4);
  const int row = job.rb * rb_rows + local;
  const bool live =
      local < rb_rows && row < a.rows && row % a.nodes < clamped_nodes(a, job.b);
  if (__ballot(live) == 0) return;
  const int at = live ? local : 0;  // (a row of the unit's, where there is one)
  const int n = static_cast<int>(blockIdx.x) - job.first + 1;
  auto slot = [&](int i) {
    return static_cast<std::size_t>(2 * (job.first + i) + (i == 0 ? 1 : 0));
  };
  float top = -INFINITY, sum = 0.f;
  v4f o[2] = {v4f{0.f, 0.f, 0.f, 0.f}, v4f{0.f, 0.f, 0.f, 0.f}};
  bool again = false;  // some part of a row of this wavefront is marked
  for (int i0 = 0; i0 < n; i0 += 16) {
    float m = -INFINITY, l = 0.f;
    bool marked = false;
    if (i0 + part < n) {
      const std::size_t s = slot(i0 + part);
      const float2 x = *reinterpret_cast<const float2*>(st.part_ml + (s * rb_rows + at) * 2);
      marked = live && st.part_marks[s * kMaxTiles + at / 16] != 0;
      if (live && !marked) {
        m = x.x;
        l = x.y;
      }
    }
    again = again || __ballot(marked) != 0;
    float mx = m;
#pragma unroll
    for (int k = 8; k > 0; k /= 2) mx = fmaxf(mx, __shfl_xor(mx, k, 64));
    const float mn = fmaxf(top, mx);
    const float alpha = exp2_ratio(top, mn);
    const float w = i0 + part < n && live && !marked ? exp2_ratio(m, mn) : 0.f;
    float add = w * l;
#pragma unroll
    for (int k = 8; k > 0; k /= 2) add += __shfl_xor(add, k, 64);
    sum = sum * alpha + add;
    o[0] *= alpha;
    o[1] *= alpha;
    top = mn;
    const int end = min(n - i0, 16);
    for (int i = 0; i < end; ++i) {
      const int from = (lane & 48) + i;
      const float wi = __shfl(w, from, 64);
      const bool skip = __shfl(marked ? 1 : 0, from, 64) != 0;
      const auto* x = reinterpret_cast<const v4f*>(st.part_o + (slot(i0 + i) * rb_rows + at) * D) +
                      2 * part;
      const v4f x0 = x[0], x1 = x[1];
      if (!skip) {
        o[0] += wi * x0;
        o[1] += wi * x1;
      }
    }
  }
  if (again) {
    // The marked parts of the wavefront's four rows, a row after another; lane
    // i of 64 holds dims 2 i, 2 i + 1 there and hands them over.
    const TreeSequence s = tree_sequence(a, job.b, lane);
    const unsigned long long broken = __ballot(s.broken != 0);
    const int nbh = (s.hist + kBlock - 1) / kBlock;
    auto tokens = [&](long long blocks) {
      return static_cast<int>(min(static_cast<long long>(s.hist), blocks * kBlock));
    };
    auto nodes = [&](long long blocks) {
      return static_cast<int>(
          min(static_cast<long long>(s.count), max(blocks - nbh, 0ll) * kBlock));
    };
#pragma unroll 1
    for (int r = 0; r < 4; ++r) {
      const int one = static_cast<int>(blockIdx.y) * kMergeRows + wave * 4 + r;
      const int one_row = job.rb * rb_rows + one;
      if (one >= rb_rows || one_row >= a.rows || one_row % a.nodes >= s.count) continue;
      if (((broken >> (one_row % a.nodes)) & 1) != 0) {
        // (Its NaN may stand in a part that is marked for the tile's other rows.)
        if (lane >> 4 == r) sum = NAN;
        continue;
      }
#pragma unroll 1
      for (int i = 0; i < n; ++i) {
        if (st.part_marks[slot(i) * kMaxTiles + one / 16] == 0) continue;
        const long long from = i == 0 ? 0 : job.head + static_cast<long long>(i - 1) * job.each;
        const long long to = job.head + static_cast<long long>(i) * job.each;
        float2 e;
        float em, el;
        exact_row<PF>(a, job.b, job.kvh, one_row, tokens(from), tokens(to), nodes(from), nodes(to),
                      shfl64(s.seen, one_row % a.nodes), lane, e, em, el);
        float d[8];  // this lane's dims, had it the row
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          d[2 * k] = __shfl(e.x, 4 * part + k, 64);
          d[2 * k + 1] = __shfl(e.y, 4 * part + k, 64);
        }
        if (lane >> 4 == r) {
          const float en = fmaxf(top, em);
          const float f = exp2_ratio(top, en);
          const float g = exp2_ratio(em, en) * (PF == 2 ? kProbScale : 1.0f);
          sum = sum * f + el * g;
          o[0] = o[0] * f + v4f{d[0], d[1], d[2], d[3]} * g;
          o[1] = o[1] * f + v4f{d[4], d[5], d[6], d[7]} * g;
          top = en;
        }
      }
    }
  }
  if (!live) return;
  const float f = top == -INFINITY ? NAN : 1.0f / sum;
  auto* const dst = reinterpret_cast<v4f*>(out_row(job.b, job.kvh, row)) + 2 * part;
  dst[0] = o[0] * f;
  dst[1] = o[1] * f;
}

// ----------------------------------------------------------------- host ----
constexpr std::size_t kTreeCus = 256;

struct TreeShape {
  int waves, tiles;      // wavefronts of a workgroup, 16-row tiles of one
  std::size_t groups;    // workgroups of a launch
  std::size_t rows() const { return static_cast<std::size_t>(waves) * tiles * 16; }
};

// A unit's rows and the workgroups that the chip holds at once.  32 sequences of 512
// to 8192 tokens, 32/8 heads, in us:
//                          bf16 pages       fp32 pages       fp8 pages
//   rows of a head       64  128  256     64  128  256     64  128  256
//   4 wavefronts        110  158  390    192  300  762     92  128  296
//   4 of two tiles        -    -    -      -    -    -    117  113  242
//   8 wavefronts        127  143  332    206  249  626      -    -    -
//   8 of two tiles      209  198  297    432  386  559      -    -    -
// (An item of fp8 pages is four jobs, of a wavefront each.)
TreeShape tree_shape(PageType type, std::size_t rows) {
  if (type == PageType::kFP8) {
    return rows <= 64 ? TreeShape{4, 1, 3 * kTreeCus} : TreeShape{4, 2, 2 * kTreeCus};
  }
  if (rows <= 64) return {4, 1, 2 * kTreeCus};
  return rows <= 128 ? TreeShape{8, 1, kTreeCus} : TreeShape{8, 2, kTreeCus};
}

std::size_t align256(std::size_t n) { return (n + 255) & ~std::size_t{255}; }

// The workspace: jobs, partials' marks, units' marks, statistics, outputs.
struct TreeLayout {
  TreeLayout(const TreeShape& s, std::size_t batch, std::size_t kv_heads, std::size_t rows) {
    row_blocks = (rows + s.rows() - 1) / s.rows();
    auto take = [&](std::size_t n) {
      const std::size_t at = bytes;
      bytes += align256(n);
      return at;
    };
    jobs = take(s.groups * sizeof(TreeJob));
    part_marks = take(2 * s.groups * kMaxTiles);
    unit_marks = take(batch * kv_heads * row_blocks * kMaxTiles);
    part_ml = take(2 * s.groups * s.rows() * 2 * sizeof(float));
    part_o = take(2 * s.groups * s.rows() * D * sizeof(float));
  }
  std::size_t row_blocks, jobs, part_marks, unit_marks, part_ml, part_o, bytes = 0;
};

template <int PF, int W, int RT>
void launch_mma(const TreeKernelArgs& k, const TreeStream& st, hipStream_t stream) {
  tree_mma_kernel<PF, W, RT>
      <<<dim3(static_cast<unsigned>(st.groups)), 64 * W, 0, stream>>>(k, st);
}

template <int PF>
hipError_t launch_tree(const TreeKernelArgs& k, const TreeStream& st, const TreeShape& s,
                       hipStream_t stream) {
  if (s.rows() == 64) {
    launch_mma<PF, 4, 1>(k, st, stream);
  } else if constexpr (PF == 2) {
    launch_mma<PF, 4, 2>(k, st, stream);
  } else if (s.rows() == 128) {
    launch_mma<PF, 8, 1>(k, st, stream);
  } else {
    launch_mma<PF, 8, 2>(k, st, stream);
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const int rows = static_cast<int>(s.rows()) < k.rows ? static_cast<int>(s.rows()) : k.rows;
  const dim3 grid(static_cast<unsigned>(st.groups),
                  static_cast<unsigned>((rows + kMergeRows - 1) / kMergeRows));
  tree_merge_kernel<PF><<<grid, 256, 0, stream>>>(k, st, static_cast<int>(s.rows()));
  return hipGetLastError();
}

}  // namespace

std::size_t tree_workspace_bytes(std::size_t batch, std::size_t q_heads, std::size_t kv_heads,
                                 std::size_t nodes) {
  const std::size_t rows = q_heads / kv_heads * nodes;
  std::size_t bytes = 0;  // for any type of page
  for (const PageType type : {PageType::kF32, PageType::kBF16, PageType::kFP8}) {
    bytes = std::max(bytes, TreeLayout(tree_shape(type, rows), batch, kv_heads, rows).bytes);
  }
  return bytes;
}

bool tree_fits(const TreeAttentionArgs& a) {
  // Ranges, and places in them, are counted in 32 bits: of 2^38 blocks, a
  // group's are 2^30 at most.  (The grid's limits keep the product in 64 bits.)
  const std::size_t rows = a.q_heads / a.kv_heads * a.nodes;
  const std::size_t units = a.batch * a.kv_heads * ((rows + 63) / 64);
  return units == 0 || a.max_blocks / 2 + 3 <= (std::size_t{1} << 38) / units;
}

hipError_t launch_tree_attention(const TreeAttentionArgs& a, hipStream_t stream) {
  if (a.batch == 0 || a.nodes == 0) return hipSuccess;
  if (!tree_fits(a)) return hipErrorInvalidValue;
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
  const TreeShape s = tree_shape(a.page_type.type, static_cast<std::size_t>(k.rows));
  const TreeLayout layout(s, a.batch, a.kv_heads, static_cast<std::size_t>(k.rows));
  auto* const base = static_cast<unsigned char*>(a.workspace);
  TreeStream st{};
  st.jobs = reinterpret_cast<TreeJob*>(base + layout.jobs);
  st.part_marks = base + layout.part_marks;
  st.unit_marks = base + layout.unit_marks;
  st.part_ml = reinterpret_cast<float*>(base + layout.part_ml);
  st.part_o = reinterpret_cast<float*>(base + layout.part_o);
  st.groups = static_cast<int>(s.groups);
  st.row_blocks = static_cast<int>(layout.row_blocks);
  switch (a.page_type.type) {
    case PageType::kBF16: return launch_tree<1>(k, st, s, stream);
    case PageType::kFP8: return launch_tree<2>(k, st, s, stream);
    default: return launch_tree<0>(k, st, s, stream);
  }
}

}  // namespace helix::hip
