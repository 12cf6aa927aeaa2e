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
//   probabilities (with them sums and outputs) carry a factor of 2^14;
// - fp32 pages: three bf16 terms on either side, less the products below
//   2^-26 of the largest: 6 products, 2.7 times the rate of fp32 matrix
//   instructions.
// Elements are split or widened once per workgroup on their way into LDS.
//
// Special values.  Terms of infinities, a 0 times an infinity and values that
// a row does not see can only show as a NaN in the row's sum or outputs.  A
// tile of 16 rows that ends a part with one is marked, and tree_merge_kernel
// computes that part of it again with exact_row.
#include "prefill_bmma.hpp"
#include "tree_exact.hpp"

#include <hip/hip_runtime.h>

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
constexpr float kProbScale = 16384.0f;  // fp8 pages

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
  int least;       // blocks of a range at least
};

// x = t[0] + t[1] (+ t[2]), each rounded to nearest; two numbers at a time,
// packed into words.
template <int PF>
__device__ __forceinline__ void split_pair(float x, float y, unsigned (&t)[3]) {
  if constexpr (PF == 2) {
    const v2h hi = {static_cast<_Float16>(x), static_cast<_Float16>(y)};
    const v2h lo = {static_cast<_Float16>(x - static_cast<float>(hi[0])),
                    static_cast<_Float16>(y - static_cast<float>(hi[1]))};
    t[0] = __builtin_bit_cast(unsigned, hi);
    t[1] = __builtin_bit_cast(unsigned, lo);
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

template <int PF>
__device__ __forceinline__ v4f matrix_step(uint4 a, uint4 b, v4f c) {
  if constexpr (PF == 2) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a),
                                                  __builtin_bit_cast(v8h, b), c, 0, 0, 0);
  } else {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a),
                                                   __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
  }
}

// Eight fp8 codes as fp16.
__device__ __forceinline__ uint4 codes_fp16(unsigned w0, unsigned w1) {
  return make_uint4(
      __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w0, 1.0f, false)),
      __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w0, 1.0f, true)),
      __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w1, 1.0f, false)),
      __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w1, 1.0f, true)));
}

// 16 bytes of each plane a chunk of 8 elements becomes in LDS: from 8 fp32
// values (a tree row, or an fp32 page), rounded onto the page grid.
template <int PF>
__device__ __forceinline__ void chunk_of_rows(v4f x0, v4f x1, float scale,
                                              uint4 (&t)[page_terms(PF)]) {
  if constexpr (PF == 0) {
    unsigned w[4][3];
    split_pair<0>(x0[0], x0[1], w[0]);
    split_pair<0>(x0[2], x0[3], w[1]);
    split_pair<0>(x1[0], x1[1], w[2]);
    split_pair<0>(x1[2], x1[3], w[3]);
#pragma unroll
    for (int i = 0; i < 3; ++i) t[i] = make_uint4(w[0][i], w[1][i], w[2][i], w[3][i]);
  } else if constexpr (PF == 1) {
    t[0] = make_uint4(bf16_pack(x0[0], x0[1]), bf16_pack(x0[2], x0[3]), bf16_pack(x1[0], x1[1]),
                      bf16_pack(x1[2], x1[3]));
  } else {
    t[0] = codes_fp16(fp8_pack4_scaled(make_float4(x0[0], x0[1], x0[2], x0[3]), scale),
                      fp8_pack4_scaled(make_float4(x1[0], x1[1], x1[2], x1[3]), scale));
  }
}

template <int PF, int TILES>
struct TreeShared {
  __align__(1024) unsigned char k[page_terms(PF)][kBlock * 2 * D];
  __align__(1024) unsigned char v[page_terms(PF)][kBlock * 2 * D];
  // The third terms of the query operands: [tile][step][lane].
  __align__(16) uint4 low[row_terms(PF) == 3 ? TILES : 1][row_terms(PF) == 3 ? 4 : 1][64];
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
__device__ __forceinline__ long long lane_scan(int v, int lane) {
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
  long long g0, g1, each;
};
__device__ __forceinline__ TreeRange first_place(const TreeKernelArgs& a, const TreeStream& st,
                                                 int group, int lane, TreeCursor& c) {
  long long per_head = 0;
  for (int b0 = 0; b0 < a.batch; b0 += 64) {
    per_head += uniform_long(__shfl(lane_scan(lane_blocks(a, b0 + lane), lane), 63, 64));
  }
  per_head *= st.row_blocks;
  const long long total = per_head * a.kv_heads;
  TreeRange r{};
  r.each = uniform_long(max((total + st.groups - 1) / st.groups, static_cast<long long>(st.least)));
  r.g0 = uniform_long(group * r.each);
  r.g1 = uniform_long(min(r.g0 + r.each, total));
  if (r.g0 >= r.g1) return r;
  c.kvh = __builtin_amdgcn_readfirstlane(static_cast<int>(r.g0 / per_head));
  const long long rem = r.g0 - c.kvh * per_head;
  long long base = 0;
  for (int b0 = 0; b0 < a.batch; b0 += 64) {
    const int nb = lane_blocks(a, b0 + lane);
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

// W wavefronts of RT tiles of 16 query rows: units of RB = 16 W RT rows.
template <int PF, int W, int RT>
__device__ __forceinline__ void tree_mma_body(const TreeKernelArgs& a, const TreeStream& st,
                                              TreeShared<PF, W * RT>& sh) {
  constexpr int NT = 64 * W;
  constexpr int NC = kBlock * D / 8 / NT;  // 8-element chunks of K (and of V) per thread
  constexpr int RB = 16 * W * RT;
  constexpr int KT = page_terms(PF), QT = row_terms(PF);
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, grp = lane >> 4;
  const int group = static_cast<int>(blockIdx.x);
  auto barrier = [] {
    if constexpr (W == 1) {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    } else {
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    }
  };

  if (tid == 0) st.jobs[group] = TreeJob{-1, 0, 0, 0, 0, 0};
  TreeCursor cur{};
  const TreeRange range = first_place(a, st, group, lane, cur);
  if (range.g0 >= range.g1) return;

  // Pages of the unit in hand, 64 at a time: lane i holds page ids_at + i.
  unsigned ids = 0;
  int ids_b = -1, ids_at = 0;
  bool bad_page = false;

  // A block's rows on their way: chunk tid + NT i, row chunk / 16.
  using Raw = std::conditional_t<PF == 0, v4f, std::conditional_t<PF == 1, v4u, v2u>>;
  constexpr int RW = PF == 0 ? 2 : 1;
  Raw kr[NC * RW], vr[NC * RW];
  auto load_block = [&](const TreeCursor& c) {
    if (c.blk >= c.nbh) return;  // tree rows are loaded when they are stored
    const int first = 2 * c.blk;
    if (ids_b != c.b || first < ids_at || first >= ids_at + 64) {
      ids_b = c.b;
      ids_at = first;
      const int last = (c.hist - 1) / P;
      ids = a.tables[static_cast<std::size_t>(c.b) * a.max_blocks + min(first + lane, last)];
    }
    // (Behind the history the last page is read again; a page outside the pool
    // is not read.)
    auto page_at = [&](int h) {
      unsigned page = __builtin_amdgcn_readlane(ids, first + h - ids_at);
      if (page >= a.physical_blocks) {
        bad_page = true;
        page = 0;
      }
      return (static_cast<std::size_t>(page) * a.kv_heads + c.kvh) * (P * D);
    };
    const std::size_t at0 = page_at(0), at1 = page_at(1);
    constexpr int kElem = PF == 0 ? 4 : PF == 1 ? 2 : 1;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int base = wave * 64 + NT * i;  // of the wavefront's chunks, in one page
      const std::size_t e = ((base >= 256 ? at1 : at0) + (base & 255) * 8) * kElem;
      const auto* k = reinterpret_cast<const Raw*>(static_cast<const unsigned char*>(a.key_pool) + e) +
                      static_cast<unsigned>(lane * RW);
      const auto* v = reinterpret_cast<const Raw*>(static_cast<const unsigned char*>(a.value_pool) + e) +
                      static_cast<unsigned>(lane * RW);
#pragma unroll
      for (int w = 0; w < RW; ++w) {
        kr[i * RW + w] = k[w];
        vr[i * RW + w] = v[w];
      }
    }
  };
  auto store_block = [&](const TreeCursor& c) {
    const bool tree = c.blk >= c.nbh;
    const int seen = tree ? c.count - (c.blk - c.nbh) * kBlock : c.hist - c.blk * kBlock;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int chunk = tid + NT * i, row = chunk >> 4, part = chunk & 15;
      uint4 kt[KT], vt[KT];
      if (tree) {
        const int node = (c.blk - c.nbh) * kBlock + min(row, seen - 1);
        const std::size_t e =
            ((static_cast<std::size_t>(c.b) * a.kv_heads + c.kvh) * a.nodes + node) * D + part * 8;
        // (Global address space, or the compiler merges these loads with reads of
        // kr and vr, which must stay in registers.)
        using Rows = const __attribute__((address_space(1))) v4f*;
        const auto k = reinterpret_cast<Rows>(reinterpret_cast<std::uintptr_t>(a.tree_key + e));
        const auto v = reinterpret_cast<Rows>(reinterpret_cast<std::uintptr_t>(a.tree_value + e));
        chunk_of_rows<PF>(k[0], k[1], a.k_scale, kt);
        chunk_of_rows<PF>(v[0], v[1], a.v_scale, vt);
      } else if constexpr (PF == 0) {
        chunk_of_rows<0>(kr[2 * i], kr[2 * i + 1], 1.0f, kt);
        chunk_of_rows<0>(vr[2 * i], vr[2 * i + 1], 1.0f, vt);
      } else if constexpr (PF == 1) {
        kt[0] = __builtin_bit_cast(uint4, kr[i]);
        vt[0] = __builtin_bit_cast(uint4, vr[i]);
      } else {
        kt[0] = codes_fp16(kr[i][0], kr[i][1]);
        vt[0] = codes_fp16(vr[i][0], vr[i][1]);
      }
#pragma unroll
      for (int t = 0; t < KT; ++t) {
        if (row >= seen) kt[t] = vt[t] = make_uint4(0u, 0u, 0u, 0u);
        *reinterpret_cast<uint4*>(sh.k[t] + bmma_k_at(row, part)) = kt[t];
        *reinterpret_cast<uint4*>(sh.v[t] + bmma_v_at(row, part)) = vt[t];
      }
    }
  };

  // The wavefront's rows of the unit: tile t's row `col`.
  uint4 qop[RT][2][4];  // (the third term of three is in LDS)
  float unscale[RT];  // fp8 pages: what undoes the row's power of two
  auto unit_rows = [&](const TreeCursor& c) {
    return (static_cast<std::size_t>(c.b) * a.q_heads +
            static_cast<std::size_t>(c.kvh) * (a.q_heads / a.kv_heads)) *
           a.nodes;
  };
  auto load_query = [&](const TreeCursor& c) {
    const float scale = PF == 2 ? a.qscale * a.k_scale : a.qscale;
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      const int row = c.rb * RB + (wave * RT + t) * 16 + col;
      float4 x[4][2];
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        x[s][0] = x[s][1] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (row < a.rows) {
          const auto* q =
              reinterpret_cast<const float4*>(a.query + (unit_rows(c) + row) * D + 32 * s + 8 * grp);
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
            most = fmaxf(most, fmaxf(fmaxf(fabsf(x[s][w].x), fabsf(x[s][w].y)),
                                     fmaxf(fabsf(x[s][w].z), fabsf(x[s][w].w))));
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
        const float y[8] = {x[s][0].x, x[s][0].y, x[s][0].z, x[s][0].w,
                            x[s][1].x, x[s][1].y, x[s][1].z, x[s][1].w};
        unsigned w[4][3];
#pragma unroll
        for (int i = 0; i < 4; ++i) split_pair<PF>(y[2 * i] * grow, y[2 * i + 1] * grow, w[i]);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          qop[t][i][s] = make_uint4(w[0][i], w[1][i], w[2][i], w[3][i]);
        }
        if constexpr (QT == 3) {
          sh.low[wave * RT + t][s][lane] = make_uint4(w[0][2], w[1][2], w[2][2], w[3][2]);
        }
      }
    }
  };

  v4f o[RT][8];  // o[t][dt][i]: dim 16 dt + 4 grp + i of row col
  float m[RT], l[RT];
  unsigned long long broken = 0;  // the nodes with a wrong parent on their way

  const unsigned k_at = bmma_k_at(col, grp);
  const unsigned v_at =
      bmma_v_at(4 * grp + (col >> 2), 0) + static_cast<unsigned>((col & 3) * 8);
  auto compute = [&](const TreeCursor& c) {
    v4f sc[RT][2];
#pragma unroll
    for (int t = 0; t < RT; ++t) sc[t][0] = sc[t][1] = v4f{0.f, 0.f, 0.f, 0.f};
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      uint4 low[RT];
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        if constexpr (QT == 3) low[t] = sh.low[wave * RT + t][s][lane];
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint4 kop[KT];
#pragma unroll
        for (int i = 0; i < KT; ++i) {
          kop[i] = *reinterpret_cast<const uint4*>(sh.k[i] + h * (P * 2 * D) + (k_at ^ (64u * s)));
        }
#pragma unroll
        for (int t = 0; t < RT; ++t) {
          // Smallest products first.
#pragma unroll
          for (int sum = QT - 1; sum >= 0; --sum) {
#pragma unroll
            for (int i = KT - 1; i >= 0; --i) {
              if (sum - i < 0 || sum - i >= QT) continue;
              sc[t][h] =
                  matrix_step<PF>(kop[i], sum - i == 2 ? low[t] : qop[t][sum - i & 1][s], sc[t][h]);
            }
          }
        }
      }
    }
    __builtin_amdgcn_s_setprio(0);
    const bool in_tree = c.blk >= c.nbh;
    const int seen = in_tree ? 0 : c.hist - c.blk * kBlock;
    unsigned bits[RT];  // the block's keys that the row sees
    if (in_tree) {
      const TreeSequence tree = tree_sequence(a, c.b, lane);
      broken = __ballot(tree.broken != 0);
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        const int row = c.rb * RB + (wave * RT + t) * 16 + col;
        const unsigned long long w = shfl64(tree.seen, row % a.nodes);
        bits[t] = row < a.rows ? static_cast<unsigned>(w >> ((c.blk - c.nbh) * kBlock)) : 0u;
      }
    } else {
#pragma unroll
      for (int t = 0; t < RT; ++t) bits[t] = seen >= kBlock ? ~0u : (1u << seen) - 1u;
    }
    uint4 pop[RT][QT];
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      // x[j]: key 16 (j / 4) + 4 grp + j % 4.
      float x[8], p[8];
      unsigned vis = 0xffu;
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = sc[t][j >> 2][j & 3];
      if constexpr (PF == 2) {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] *= unscale[t];
      }
      const bool full = !in_tree && seen >= kBlock;
      if (!full) {
        vis = ((bits[t] >> (4 * grp)) & 0xfu) | ((bits[t] >> (16 + 4 * grp)) & 0xfu) << 4;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (((vis >> j) & 1u) == 0) x[j] = -INFINITY;
        }
      }
      const float mx = row_max(fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])),
                                     fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7]))));
      const float mn = fmaxf(m[t], mx);
      if (__ballot(!(mn == m[t])) != 0) {  // some row's maximum moved
        const float alpha = exp2_ratio(m[t], mn);
#pragma unroll
        for (int dt = 0; dt < 8; ++dt) o[t][dt] *= alpha;
        l[t] *= alpha;
        m[t] = mn;
      }
      if (full && __ballot(!(fabsf(mn) < INFINITY)) == 0) {
        const float shift = PF == 2 ? mn - 14.0f : mn;
#pragma unroll
        for (int j = 0; j < 8; ++j) p[j] = __builtin_amdgcn_exp2f(x[j] - shift);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          p[j] = ((vis >> j) & 1u) != 0 ? exp2_ratio(x[j], mn) : 0.f;
          if constexpr (PF == 2) p[j] *= kProbScale;
        }
      }
      // The lane's own keys; the row's four lanes are added at the end.
      l[t] += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
      unsigned w[4][3];
#pragma unroll
      for (int i = 0; i < 4; ++i) split_pair<PF>(p[2 * i], p[2 * i + 1], w[i]);
#pragma unroll
      for (int i = 0; i < QT; ++i) pop[t][i] = make_uint4(w[0][i], w[1][i], w[2][i], w[3][i]);
    }
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int dt = 0; dt < 8; ++dt) {
      using LdsV4s = __attribute__((address_space(3))) v4s;
      uint4 vop[KT];
#pragma unroll
      for (int i = 0; i < KT; ++i) {
        const unsigned char* vp = sh.v[i] + (v_at ^ (32u * dt));
        const v4s v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsV4s*)(vp));
        const v4s v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsV4s*)(vp + P * 2 * D));
        vop[i] = __builtin_bit_cast(uint4, __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7));
      }
#pragma unroll
      for (int t = 0; t < RT; ++t) {
#pragma unroll
        for (int sum = QT - 1; sum >= 0; --sum) {
#pragma unroll
          for (int i = KT - 1; i >= 0; --i) {
            if (sum - i < 0 || sum - i >= QT) continue;
            o[t][dt] = matrix_step<PF>(vop[i], pop[t][sum - i], o[t][dt]);
          }
        }
      }
    }
    __builtin_amdgcn_s_setprio(0);
  };

  // Ends the unit's part [from, c.blk] in this range.
  auto finish = [&](const TreeCursor& c, int from, long long g) {
    const bool starts = from == 0, ends = c.blk + 1 == c.nb;
    const bool complete = starts && ends;
    const float vscale = PF == 2 ? a.v_scale : 1.0f;
    const bool bad = bad_page || c.bad;
    bad_page = false;
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
      const int row = c.rb * RB + (wave * RT + t) * 16 + col, node = row % a.nodes;
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
        marks[wave * RT + t] = again ? 1 : 0;
        if (ends && !starts) st.unit_marks[unit * kMaxTiles + wave * RT + t] = 0;
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

  load_block(cur);
  int from = cur.blk;  // the unit's first block in this range
  bool fresh = true;
  for (long long g = range.g0;; ++g) {
    barrier();
    store_block(cur);
    barrier();
    const bool more = g + 1 < range.g1;
    if (fresh) {
      load_query(cur);
#pragma unroll
      for (int t = 0; t < RT; ++t) {
#pragma unroll
        for (int dt = 0; dt < 8; ++dt) o[t][dt] = v4f{0.f, 0.f, 0.f, 0.f};
        m[t] = -INFINITY;
        l[t] = 0.f;
      }
      fresh = false;
      broken = 0;
    }
    const bool bad_before = bad_page;
    bad_page = false;
    TreeCursor next = cur;
    if (more) {
      advance(a, st, next);
      load_block(next);
    }
    const bool bad_next = bad_page;
    bad_page = bad_before;
    compute(cur);
    if (!more || cur.blk + 1 == cur.nb) {
      finish(cur, from, g);
      from = 0;
      fresh = true;
    }
    bad_page = bad_page || bad_next;
    if (!more) break;
    cur = next;
  }
}

template <int PF, int W, int RT>
__global__ __launch_bounds__(64 * W) __attribute__((amdgpu_waves_per_eu(PF == 0 ? (W == 1 ? 1 : 2) : W <= 2 || RT == 2 ? 2 : 3))) void tree_mma_kernel(TreeKernelArgs a, TreeStream st) {
  __shared__ TreeShared<PF, W * RT> sh;
  tree_mma_body<PF, W, RT>(a, st, sh);
}

// Joins the partials of the units that cross ranges: blockIdx.x is the group
// whose range ends such a unit, its partials the first group's second slot and
// the later groups' first ones.  A wavefront takes a row, a lane two dims.
// Marked parts are computed again here; those of finished units by the
// workgroups with blockIdx.y = 0.
constexpr int kMergeRows = 4;
template <int PF>
__global__ __launch_bounds__(64 * kMergeRows) void tree_merge_kernel(TreeKernelArgs a,
                                                                     TreeStream st, int rb_rows) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  auto out_row = [&](int b, int kvh, int row) {
    return reinterpret_cast<float2*>(
               a.out + ((static_cast<std::size_t>(b) * a.q_heads +
                         static_cast<std::size_t>(kvh) * (a.q_heads / a.kv_heads)) * a.nodes +
                        row) * D) + lane;
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
      for (int i = wave; i < rb_rows; i += kMergeRows) {
        const int row = rb * rb_rows + i, node = row % a.nodes;
        if (st.unit_marks[u * kMaxTiles + i / 16] == 0 || row >= a.rows || node >= s.count) continue;
        if (((__ballot(s.broken != 0) >> node) & 1) != 0) continue;
        float2 o;
        float m, l;
        exact_row<PF>(a, b, kvh, row, 0, s.hist, 0, s.count, shfl64(s.seen, node), lane, o, m, l);
        const float f = m == -INFINITY ? NAN : 1.0f / l;
        *out_row(b, kvh, row) = make_float2(o.x * f, o.y * f);
      }
    }
  }
  const TreeJob job = st.jobs[blockIdx.x];
  if (job.b < 0) return;
  const int local = static_cast<int>(blockIdx.y) * kMergeRows + wave;
  const int row = job.rb * rb_rows + local;
  if (local >= rb_rows || row >= a.rows || row % a.nodes >= clamped_nodes(a, job.b)) return;
  const int n = static_cast<int>(blockIdx.x) - job.first + 1;
  auto slot = [&](int i) {
    return static_cast<std::size_t>(2 * (job.first + i) + (i == 0 ? 1 : 0));
  };
  float top = -INFINITY, sum = 0.f;
  float2 o = make_float2(0.f, 0.f);
  for (int i0 = 0; i0 < n; i0 += 64) {
    float m = -INFINITY, l = 0.f;
    bool again = false;
    if (i0 + lane < n) {
      const std::size_t at = slot(i0 + lane);
      const float2 x = *reinterpret_cast<const float2*>(st.part_ml + (at * rb_rows + local) * 2);
      again = st.part_marks[at * kMaxTiles + local / 16] != 0;
      if (!again) {
        m = x.x;
        l = x.y;
      }
    }
    float mx = m;
#pragma unroll
    for (int k = 32; k > 0; k /= 2) mx = fmaxf(mx, __shfl_xor(mx, k, 64));
    const float mn = fmaxf(top, mx);
    const float alpha = exp2_ratio(top, mn);
    const float w = i0 + lane < n && !again ? exp2_ratio(m, mn) : 0.f;
    float add = w * l;
#pragma unroll
    for (int k = 32; k > 0; k /= 2) add += __shfl_xor(add, k, 64);
    sum = sum * alpha + add;
    o.x *= alpha;
    o.y *= alpha;
    top = mn;
    unsigned long long marked = __ballot(again);
    const int end = min(n - i0, 64);
    for (int i = 0; i < end; ++i) {
      if (((marked >> i) & 1) != 0) continue;
      const float wi = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(w), i));
      const float2 x = *reinterpret_cast<const float2*>(
          st.part_o + (slot(i0 + i) * rb_rows + local) * D + 2 * lane);
      o.x += wi * x.x;
      o.y += wi * x.y;
    }
    for (; marked != 0; marked &= marked - 1) {
      const int i = i0 + __ffsll(static_cast<long long>(marked)) - 1;
      const TreeSequence s = tree_sequence(a, job.b, lane);
      const int nbh = (s.hist + kBlock - 1) / kBlock;
      const long long from = i == 0 ? 0 : job.head + static_cast<long long>(i - 1) * job.each;
      const long long to = job.head + static_cast<long long>(i) * job.each;
      auto tokens = [&](long long blocks) {
        return static_cast<int>(min(static_cast<long long>(s.hist), blocks * kBlock));
      };
      auto nodes = [&](long long blocks) {
        return static_cast<int>(min(static_cast<long long>(s.count), max(blocks - nbh, 0ll) * kBlock));
      };
      float2 e;
      float em, el;
      exact_row<PF>(a, job.b, job.kvh, row, tokens(from), tokens(to), nodes(from), nodes(to),
                    shfl64(s.seen, row % a.nodes), lane, e, em, el);
      const float en = fmaxf(top, em);
      const float f = exp2_ratio(top, en), g = exp2_ratio(em, en) * (PF == 2 ? kProbScale : 1.0f);
      sum = sum * f + el * g;
      o.x = o.x * f + e.x * g;
      o.y = o.y * f + e.y * g;
      top = en;
    }
  }
  const float f = top == -INFINITY ? NAN : 1.0f / sum;
  *out_row(job.b, job.kvh, row) = make_float2(o.x * f, o.y * f);
}

// ----------------------------------------------------------------- host ----
constexpr std::size_t kTreeCus = 256;

struct TreeShape {
  int waves, tiles;      // wavefronts of a workgroup, 16-row tiles of one
  std::size_t groups;    // workgroups of a launch
  std::size_t rows() const { return static_cast<std::size_t>(waves) * tiles * 16; }
};

TreeShape tree_shape(std::size_t rows) {
  const std::size_t tiles = (rows + 15) / 16;
  if (tiles <= 1) return {1, 1, 4 * kTreeCus};
  if (tiles <= 2) return {2, 1, 3 * kTreeCus};
  if (tiles <= 4) return {4, 1, 2 * kTreeCus};
  if (tiles <= 8) return {4, 2, 2 * kTreeCus};
  return {8, 2, kTreeCus};
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
  switch (s.waves * 10 + s.tiles) {
    case 11: launch_mma<PF, 1, 1>(k, st, stream); break;
    case 21: launch_mma<PF, 2, 1>(k, st, stream); break;
    case 41: launch_mma<PF, 4, 1>(k, st, stream); break;
    case 42: launch_mma<PF, 4, 2>(k, st, stream); break;
    case 82: launch_mma<PF, 8, 2>(k, st, stream); break;
    default: return hipErrorInvalidValue;
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const int rows = static_cast<int>(s.rows()) < k.rows ? static_cast<int>(s.rows()) : k.rows;
  const dim3 grid(static_cast<unsigned>(st.groups),
                  static_cast<unsigned>((rows + kMergeRows - 1) / kMergeRows));
  tree_merge_kernel<PF><<<grid, 64 * kMergeRows, 0, stream>>>(k, st, static_cast<int>(s.rows()));
  return hipGetLastError();
}

}  // namespace

std::size_t tree_workspace_bytes(std::size_t batch, std::size_t q_heads, std::size_t kv_heads,
                                 std::size_t nodes) {
  const std::size_t rows = q_heads / kv_heads * nodes;
  return TreeLayout(tree_shape(rows), batch, kv_heads, rows).bytes;
}

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
  const TreeShape s = tree_shape(static_cast<std::size_t>(k.rows));
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
  st.least = 4;
  switch (a.page_type.type) {
    case PageType::kBF16: return launch_tree<1>(k, st, s, stream);
    case PageType::kFP8: return launch_tree<2>(k, st, s, stream);
    default: return launch_tree<0>(k, st, s, stream);
  }
}

}  // namespace helix::hip
