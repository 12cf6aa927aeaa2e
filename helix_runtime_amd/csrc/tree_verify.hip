// Verification of drafted tokens: which of a tree's nodes the target's
// probabilities accept, by given random numbers, and the token that follows.
//
// For one sequence, from node n = 0 with w = p_n (the target's row at n): the
// children of n are tried in order.  Child c with token x was drawn from q_n;
// it is accepted where u_c q_n(x) < w(x), and becomes n.  Otherwise
//
//   w <- max(w - q_n, 0) / sum max(w - q_n, 0),
//
// and the next child is tried.  Without a drafter's rows, q_n is 1 on the
// child's token, and the same rule reads: accepted where u_c m < w(x), with
// m = 1 - the sum of the p_n of the tokens rejected before; a rejected token's
// w becomes 0.  Where no child is left, the following token is the smallest v
// with w(0) + .. + w(v) > bonus * sum w.  What leaves this way is distributed
// as the target's own samples.
//
// After i rejections w = max(p - c_i q, 0) / S_i with c_i = c_(i-1) + S_(i-1)
// and S_i = sum max(p - c_i q, 0) (c_0 = 0, S_0 = 1): an entry that is 0 stays
// 0, and for the others the differences add up.  So a rejection takes one sum
// over the vocabulary, of the rows as they are, and the last one's sums are
// those that the following token is chosen by.
//
// Work split.  The sums are what there is to read: a row of p and of q (1 MB at
// a vocabulary of 128256) per rejection, one after another.  A launch of
// verify_pass_kernel takes every sequence to its next sum, and computes it in
// chunks, a wavefront each; all wavefronts of a sequence make the same walk over
// the tree, of one lane per node, from what the launch before has left.  Of
// these launches there are a few.  verify_finish_kernel, a workgroup per
// sequence, takes what sums are left and chooses the token.  Nothing waits for
// another workgroup, and no result depends on an order of atomics.
//
// Sums and comparisons are 64-bit: a token hangs on each of them.
//
// Measured at a vocabulary of 128256, 64 trees of 16 nodes: the most likely tokens
// 18 us (the sum 12, 2.7 TB/s behind a walk of two dependent loads), sampled ones
// 46 (the first sum 15, 4.4 TB/s, the next ones 10 from the cache behind HBM); one
// chain of 6 at 32000 14 us, two launches of 5.
#include "tree.hpp"

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

namespace helix::hip {
namespace {

constexpr int kPassWaves = 4;
constexpr int kFinishThreads = 1024;
constexpr int kMostChunks = 64;

struct Partial {
  double sum;
  int last;  // the last entry of positive weight, or -1
  int pad;
};

// Where a sequence stands before a launch.
struct Walk {
  unsigned long long path;  // accepted nodes
  unsigned long long gone;  // rejected children of node `at`
  double c, s;              // c_i, S_i there
  double mass;
  int at, child;            // the next child to try is `child` or behind it
  int settled;              // no child is left: w is that of the token to follow
  int slot;                 // the launch that left its sums
};

struct VerifyKernelArgs {
  const float* target;
  const float* draft;
  long long target_batch_stride, target_node_stride, draft_batch_stride, draft_node_stride;
  const std::int32_t* tokens;
  const std::int32_t* parents;
  const std::int32_t* node_counts;
  const float* uniforms;
  const float* bonus_uniforms;
  std::int32_t* path;
  std::int32_t* accepted;
  std::int32_t* next_token;
  Walk* walks;        // [passes, batch]
  Partial* partials;  // [passes, batch, chunks]
  int batch, nodes, vocab;
  int chunks, chunk;  // chunks of a row, entries of one
  int passes;
};

__device__ __forceinline__ double positive(double x) { return x > 0.0 ? x : 0.0; }

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
  for (int o = 32; o > 0; o /= 2) v += __shfl_xor(v, o, 64);
  return v;
}

__device__ __forceinline__ int wave_last(int v) {
#pragma unroll
  for (int o = 32; o > 0; o /= 2) v = max(v, __shfl_xor(v, o, 64));
  return v;
}

// A sequence's tree, node `lane`: only nodes behind their parent, with a token
// of the vocabulary, can be reached; others have no parent.
struct Node {
  int parent, token;
  double u, p, q;
};
__device__ __forceinline__ Node load_node(const VerifyKernelArgs& a, int b, int count, int lane) {
  Node n{-1, -1, 0.0, 0.0, 0.0};
  if (lane >= count) return n;
  const std::size_t at = static_cast<std::size_t>(b) * a.nodes + lane;
  const int parent = a.parents != nullptr ? a.parents[at] : lane - 1;
  n.token = a.tokens[at];
  n.u = static_cast<double>(a.uniforms[at]);
  if (parent < 0 || parent >= lane || n.token < 0 || n.token >= a.vocab) return n;
  n.parent = parent;
  n.p = static_cast<double>(
      a.target[b * a.target_batch_stride + parent * a.target_node_stride + n.token]);
  if (a.draft != nullptr) {
    n.q = static_cast<double>(
        a.draft[b * a.draft_batch_stride + parent * a.draft_node_stride + n.token]);
  }
  return n;
}

// On to the next rejection whose sum is needed, or to the end (`settled`).
// Returns whether w has no sums yet.
__device__ __forceinline__ bool walk_on(const VerifyKernelArgs& a, const Node& n, int lane,
                                        Walk& w) {
  bool fresh = w.slot < 0;
  for (;;) {
    const unsigned long long left =
        __ballot(n.parent == w.at) & (w.child < 64 ? ~0ull << w.child : 0ull);
    if (left == 0) {
      w.settled = 1;
      return fresh;
    }
    const int c = __ffsll(static_cast<long long>(left)) - 1;
    w.child = c + 1;
    const int x = __shfl(n.token, c, 64);
    const double u = __shfl(n.u, c, 64), p = __shfl(n.p, c, 64), q = __shfl(n.q, c, 64);
    double weight = positive(p), need = u * w.mass;
    if (a.draft != nullptr) {
      need = u * q;
      if (w.gone != 0) weight = positive(p - w.c * q);
      if (w.s > 0.0) weight /= w.s;
    } else if ((__ballot(n.token == x) & w.gone) != 0) {
      weight = 0.0;
    }
    fresh = true;
    if (need < weight) {
      w.at = c;
      w.path |= 1ull << c;
      w.gone = 0;
      w.c = 0.0;
      w.s = w.mass = 1.0;
      continue;
    }
    w.gone |= 1ull << c;
    w.mass -= weight;
    w.c += w.s;
    if (a.draft != nullptr) return true;
  }
}

// The row that is left, entry by entry.
struct Residual {
  const float* p;
  const float* q;  // nullptr: tokens `gone` have weight 0 instead
  double c;
  __device__ __forceinline__ double at(float x, float y) const {
    const double w = static_cast<double>(x);
    return positive(q != nullptr ? w - c * static_cast<double>(y) : w);
  }
};

__device__ __forceinline__ Residual residual(const VerifyKernelArgs& a, int b, const Walk& w) {
  Residual r{a.target + b * a.target_batch_stride + w.at * a.target_node_stride, nullptr, w.c};
  if (a.draft != nullptr && w.gone != 0) {
    r.q = a.draft + b * a.draft_batch_stride + w.at * a.draft_node_stride;
  }
  return r;
}

// Four entries of a row, which need not be aligned to more than one.
__device__ __forceinline__ float4 four(const float* p) {
  float4 x;
  __builtin_memcpy(&x, p, sizeof(x));
  return x;
}

// Sum and last entry of a chunk, by a wavefront.
__device__ __forceinline__ Partial chunk_sum(const VerifyKernelArgs& a, const Residual& r,
                                             const Walk& w, const Node& n, int chunk, int lane) {
  const int begin = min(chunk * a.chunk, a.vocab), end = min(begin + a.chunk, a.vocab);
  const int token = n.token;
  // Without a drafter's rows: the rejected nodes whose tokens are in here.
  unsigned long long gone = a.draft == nullptr ? w.gone : 0;
  gone &= __ballot(token >= begin && token < end);
  double part[4] = {0.0, 0.0, 0.0, 0.0};
  int last = -1;
  auto add = [&](int v, float4 x, float4 y) {
    for (unsigned long long m = gone; m != 0; m &= m - 1) {
      const int t = __builtin_amdgcn_readlane(token, __ffsll(static_cast<long long>(m)) - 1);
      if (t == v) x.x = 0.f;
      if (t == v + 1) x.y = 0.f;
      if (t == v + 2) x.z = 0.f;
      if (t == v + 3) x.w = 0.f;
    }
    const double w0 = r.at(x.x, y.x), w1 = r.at(x.y, y.y), w2 = r.at(x.z, y.z), w3 = r.at(x.w, y.w);
    part[0] += w0;
    part[1] += w1;
    part[2] += w2;
    part[3] += w3;
    if (w0 > 0.0) last = v;
    if (w1 > 0.0) last = v + 1;
    if (w2 > 0.0) last = v + 2;
    if (w3 > 0.0) last = v + 3;
  };
  constexpr int kAhead = 4, kLanes = 4 * 64;
  int v = begin + 4 * lane;
  for (; v + kLanes * (kAhead - 1) + 4 <= end; v += kLanes * kAhead) {
    float4 x[kAhead], y[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) x[i] = four(r.p + v + kLanes * i);
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      y[i] = r.q != nullptr ? four(r.q + v + kLanes * i) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) add(v + kLanes * i, x[i], y[i]);
  }
  for (; v < end; v += kLanes) {
    float x[4], y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[i] = v + i < end ? r.p[v + i] : 0.f;
      y[i] = v + i < end && r.q != nullptr ? r.q[v + i] : 0.f;
    }
    add(v, make_float4(x[0], x[1], x[2], x[3]), make_float4(y[0], y[1], y[2], y[3]));
  }
  return Partial{wave_sum64((part[0] + part[1]) + (part[2] + part[3])), wave_last(last), 0};
}

__device__ __forceinline__ int clamped_count(const VerifyKernelArgs& a, int b) {
  return a.node_counts != nullptr ? min(max(a.node_counts[b], 0), a.nodes) : a.nodes;
}

// A wavefront's state of sequence b before launch `pass`, its sums included;
// every lane has the same.
__device__ __forceinline__ Walk load_walk(const VerifyKernelArgs& a, int b, int pass, int lane) {
  if (pass == 0) return Walk{1, 0, 0.0, 1.0, 1.0, 0, 1, 0, -1};
  Walk w = a.walks[static_cast<std::size_t>(pass - 1) * a.batch + b];
  if (w.settled == 0) {
    const Partial* const from =
        a.partials + (static_cast<std::size_t>(w.slot) * a.batch + b) * a.chunks;
    w.s = wave_sum64(lane < a.chunks ? from[lane].sum : 0.0);
  }
  return w;
}

__global__ __launch_bounds__(64 * kPassWaves) void verify_pass_kernel(VerifyKernelArgs a,
                                                                      int pass) {
  const int b = blockIdx.x, lane = threadIdx.x & 63;
  const int chunk = __builtin_amdgcn_readfirstlane(
      static_cast<int>(blockIdx.y * kPassWaves + (threadIdx.x >> 6)));
  const int count = clamped_count(a, b);
  if (count == 0 || chunk >= a.chunks) return;
  const Node n = load_node(a, b, count, lane);
  Walk w = load_walk(a, b, pass, lane);
  const bool fresh = w.settled == 0 && walk_on(a, n, lane, w);
  if (fresh) w.slot = pass;
  if (chunk == 0 && lane == 0) a.walks[static_cast<std::size_t>(pass) * a.batch + b] = w;
  if (!fresh) return;
  const Partial sum = chunk_sum(a, residual(a, b, w), w, n, chunk, lane);
  if (lane == 0) {
    a.partials[(static_cast<std::size_t>(pass) * a.batch + b) * a.chunks + chunk] = sum;
  }
}

// The first of up to 64 parts, one a lane, at whose end the running sum is above
// the goal; rounding may leave the goal behind all of them, and then it is the
// last with a weight.  `before`: the running sum there.
__device__ __forceinline__ int choose(double sum, bool any, double goal, int lane, double& before) {
  double run = sum;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double t = __shfl_up(run, o, 64);
    if (lane >= o) run += t;
  }
  double behind = __shfl_up(run, 1, 64);
  if (lane == 0) behind = 0.0;
  const unsigned long long hits = __ballot(any && before + run > goal), some = __ballot(any);
  const int at = hits != 0 ? __ffsll(static_cast<long long>(hits)) - 1
                           : 63 - __clzll(static_cast<long long>(some));
  before += __shfl(behind, at, 64);
  return at;
}

__global__ __launch_bounds__(kFinishThreads) void verify_finish_kernel(VerifyKernelArgs a) {
  constexpr int kWaves = kFinishThreads / 64;
  __shared__ Partial parts[kMostChunks];
  __shared__ Partial pieces[kWaves];
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const std::size_t row0 = static_cast<std::size_t>(b) * a.nodes;
  const int count = clamped_count(a, b);
  if (count == 0) {
    if (tid < a.nodes) a.path[row0 + tid] = -1;
    if (tid == 0) {
      a.accepted[b] = 0;
      a.next_token[b] = -1;
    }
    return;
  }
  // (Every wavefront makes the walk.)
  const Node n = load_node(a, b, count, lane);
  Walk w = load_walk(a, b, a.passes, lane);
  Partial mine{0.0, -1, 0};  // chunk `lane`
  if (w.slot >= 0 && lane < a.chunks) {
    mine = a.partials[(static_cast<std::size_t>(w.slot) * a.batch + b) * a.chunks + lane];
  }
  bool fresh = w.settled == 0 && walk_on(a, n, lane, w);
  double total;
  for (;;) {
    if (fresh) {
      const Residual r = residual(a, b, w);
      __syncthreads();
      for (int i = wave; i < a.chunks; i += kWaves) {
        const Partial sum = chunk_sum(a, r, w, n, i, lane);
        if (lane == 0) parts[i] = sum;
      }
      __syncthreads();
      mine = Partial{0.0, -1, 0};
      if (lane < a.chunks) mine = parts[lane];
      w.slot = a.passes;
    }
    total = wave_sum64(mine.sum);
    if (w.settled == 0) {
      w.s = total;
      fresh = walk_on(a, n, lane, w);
    } else if (!(total > 0.0) && w.gone != 0) {
      // Rounding left nothing of the row: its own probabilities stand.
      w.gone = 0;
      fresh = true;
    } else {
      break;
    }
  }
  int next = -1;
  if (total > 0.0) {
    const double goal = static_cast<double>(a.bonus_uniforms[b]) * total;
    double before = 0.0;
    const int chunk = choose(mine.sum, mine.last >= 0, goal, lane, before);
    // The chunk's pieces, one a wavefront, and their lanes' entries.
    const Residual r = residual(a, b, w);
    const unsigned long long gone = a.draft == nullptr ? w.gone : 0;
    const int begin = chunk * a.chunk, end = min(begin + a.chunk, a.vocab);
    const int each = (a.chunk + kFinishThreads - 1) / kFinishThreads;  // of a lane
    auto entry = [&](int v) {
      double x = r.at(r.p[v], r.q != nullptr ? r.q[v] : 0.f);
      for (unsigned long long m = gone; m != 0; m &= m - 1) {
        const int t = __builtin_amdgcn_readlane(n.token, __ffsll(static_cast<long long>(m)) - 1);
        if (t == v) x = 0.0;
      }
      return x;
    };
    const int from = begin + tid * each, to = min(from + each, end);
    double sum = 0.0;
    bool any = false;
    for (int i = 0; i < each; ++i) {
      const double x = from + i < to ? entry(from + i) : 0.0;
      sum += x;
      any = any || x > 0.0;
    }
    const double whole = wave_sum64(sum);
    const bool some = __ballot(any) != 0;
    if (lane == 0) pieces[wave] = Partial{whole, some ? 0 : -1, 0};
    __syncthreads();
    Partial piece{0.0, -1, 0};
    if (lane < kWaves) piece = pieces[lane];
    const int hit = choose(piece.sum, piece.last >= 0, goal, lane, before);
    if (wave == hit) {
      const int at = choose(sum, any, goal, lane, before);
      if (lane == at) {
        double run = before;
        for (int v = from; v < to; ++v) {
          const double x = entry(v);
          run += x;
          if (x > 0.0) next = v;
          if (x > 0.0 && run > goal) break;
        }
        a.next_token[b] = next;
      }
    }
  } else if (tid == 0) {
    a.next_token[b] = -1;
  }
  // The accepted nodes in order (a parent is before its children).
  if (wave == 0) {
    const int number = __popcll(w.path);
    if (((w.path >> lane) & 1) != 0) {
      a.path[row0 + __popcll(w.path & ((1ull << lane) - 1))] = lane;
    }
    if (lane >= number && lane < a.nodes) a.path[row0 + lane] = -1;
    if (lane == 0) a.accepted[b] = number;
  }
}

// The launches of a call and their grid.
struct VerifyShape {
  std::size_t passes, chunks, chunk;
  VerifyShape(std::size_t batch, std::size_t nodes, std::size_t vocab, bool many) {
    // About 4096 wavefronts, of at least 512 entries.
    const std::size_t most = std::clamp<std::size_t>(4096 / batch, kPassWaves, kMostChunks);
    chunks = std::max<std::size_t>(std::min(most, (vocab + 511) / 512), 1);
    chunk = ((vocab + chunks - 1) / chunks + 3) / 4 * 4;
    // A chain has one sum, as a rejection ends its walk, and so have trees
    // without a drafter's rows.  Of others, 64 trees of 16 nodes at a vocabulary
    // of 128256 take 41 us with three such launches and 44 with four where three
    // are enough, 64 and 50 where they are not: one that finds nothing to do
    // takes 2.5 us, a sum left to verify_finish_kernel 15, or less by the
    // vocabulary (one tree of 6 at 32000: 21 us with one launch, 28 with four).
    passes = 1;
    if (many) passes = std::clamp<std::size_t>(std::min(nodes - 1, (vocab + 16384) / 32768), 1, 4);
  }
  std::size_t walk_bytes(std::size_t batch) const { return passes * batch * sizeof(Walk); }
  std::size_t bytes(std::size_t batch) const {
    return walk_bytes(batch) + passes * batch * chunks * sizeof(Partial);
  }
};

}  // namespace

std::size_t verify_workspace_bytes(std::size_t batch, std::size_t nodes, std::size_t vocab) {
  if (batch == 0 || nodes == 0) return 0;
  return VerifyShape(batch, nodes, vocab, true).bytes(batch);
}

hipError_t launch_verify(const VerifyArgs& a, hipStream_t stream) {
  if (a.batch == 0 || a.nodes == 0) return hipSuccess;
  const VerifyShape shape(a.batch, a.nodes, a.vocab, a.draft != nullptr && a.parents != nullptr);
  VerifyKernelArgs k{};
  k.target = a.target;
  k.draft = a.draft;
  k.target_batch_stride = static_cast<long long>(a.target_batch_stride);
  k.target_node_stride = static_cast<long long>(a.target_node_stride);
  k.draft_batch_stride = static_cast<long long>(a.draft_batch_stride);
  k.draft_node_stride = static_cast<long long>(a.draft_node_stride);
  k.tokens = a.tokens;
  k.parents = a.parents;
  k.node_counts = a.node_counts;
  k.uniforms = a.uniforms;
  k.bonus_uniforms = a.bonus_uniforms;
  k.path = a.path;
  k.accepted = a.accepted;
  k.next_token = a.next_token;
  k.walks = static_cast<Walk*>(a.workspace);
  k.partials = reinterpret_cast<Partial*>(static_cast<unsigned char*>(a.workspace) +
                                          shape.walk_bytes(a.batch));
  k.batch = static_cast<int>(a.batch);
  k.nodes = static_cast<int>(a.nodes);
  k.vocab = static_cast<int>(a.vocab);
  k.chunks = static_cast<int>(shape.chunks);
  k.chunk = static_cast<int>(shape.chunk);
  k.passes = static_cast<int>(shape.passes);
  for (int pass = 0; pass < k.passes; ++pass) {
    verify_pass_kernel<<<dim3(static_cast<unsigned>(k.batch),
                              static_cast<unsigned>((k.chunks + kPassWaves - 1) / kPassWaves)),
                         64 * kPassWaves, 0, stream>>>(k, pass);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  verify_finish_kernel<<<dim3(static_cast<unsigned>(k.batch)), kFinishThreads, 0, stream>>>(k);
  return hipGetLastError();
}

}  // namespace helix::hip
