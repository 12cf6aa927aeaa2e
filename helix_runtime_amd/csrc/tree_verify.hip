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
// Sums and comparisons are 64-bit: a token hangs on each of them.
#include "tree.hpp"

#include <hip/hip_runtime.h>

#include <cstdint>

namespace helix::hip {
namespace {

constexpr int kVerifyThreads = 1024;
constexpr int kVerifyWaves = kVerifyThreads / 64;
constexpr int kNodes = static_cast<int>(kMaxTreeNodes);

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
  int nodes, vocab;
};

__device__ __forceinline__ double positive(double x) { return x > 0.0 ? x : 0.0; }

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
  for (int o = 32; o > 0; o /= 2) v += __shfl_xor(v, o, 64);
  return v;
}

// The row that is left at a node after some of its children were rejected.
struct Residual {
  const float* p;
  const float* q;         // nullptr: tokens `gone` have weight 0 instead
  const double* totals;   // sums of the residuals so far
  const int* gone;
  int rejected;
  // Weight of entry v; `last_raw`: the newest residual not divided by its sum.
  __device__ __forceinline__ double at(int v, bool last_raw) const {
    double w = static_cast<double>(p[v]);
    if (q == nullptr) {
      for (int i = 0; i < rejected; ++i) w = gone[i] == v ? 0.0 : w;
      return positive(w);
    }
    if (rejected == 0) return positive(w);
    const double d = static_cast<double>(q[v]);
    for (int i = 0; i < rejected; ++i) {
      w = positive(w - d);
      if ((i + 1 < rejected || !last_raw) && totals[i] > 0.0) w /= totals[i];
    }
    return w;
  }
};

struct VerifyShared {
  int parent[kNodes], token[kNodes], gone[kNodes], path[kNodes];
  double u[kNodes], p[kNodes], q[kNodes], totals[kNodes];
  double part[kVerifyWaves];
  int last[kVerifyWaves];
};

// Sums of the row's kVerifyWaves equal ranges of [from, to) into s.part, and
// each range's last entry of positive weight (or -1) into s.last.
__device__ __forceinline__ void range_sums(const Residual& r, bool raw, int from, int to,
                                           VerifyShared& s) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int each = (to - from + kVerifyWaves - 1) / kVerifyWaves;
  const int begin = from + min(wave * each, to - from);
  const int end = min(begin + each, to);
  double sum = 0.0;
  int last = -1;
  for (int v = begin + lane; v < end; v += 64) {
    const double w = r.at(v, raw);
    sum += w;
    if (w > 0.0) last = v;
  }
  sum = wave_sum64(sum);
#pragma unroll
  for (int o = 32; o > 0; o /= 2) last = max(last, __shfl_xor(last, o, 64));
  __syncthreads();
  if (lane == 0) {
    s.part[wave] = sum;
    s.last[wave] = last;
  }
  __syncthreads();
}

// The smallest v with sum of w(0) .. w(v) > bonus * total, or -1 where no
// weight is positive.
__device__ __forceinline__ int pick(const Residual& r, double bonus, int vocab, VerifyShared& s) {
  int from = 0, to = vocab;
  double before = 0.0, goal = 0.0;
  bool first = true;
  for (;;) {
    range_sums(r, false, from, to, s);
    if (first) {
      double total = 0.0;
      for (int i = 0; i < kVerifyWaves; ++i) total += s.part[i];
      if (!(total > 0.0)) return -1;
      goal = bonus * total;
      first = false;
    }
    const int each = (to - from + kVerifyWaves - 1) / kVerifyWaves;
    int hit = -1, last = -1;
    double sum = before;
    for (int i = 0; i < kVerifyWaves; ++i) {
      if (s.last[i] < 0) continue;
      last = i;  // where rounding leaves the goal behind every sum
      if (hit < 0 && sum + s.part[i] > goal) {
        hit = i;
        before = sum;
      }
      sum += s.part[i];
    }
    if (hit < 0) {
      hit = last;
      before = sum - s.part[last];
    }
    if (each == 1) return s.last[hit];
    const int next = from + hit * each;
    to = min(next + each, to);
    from = next;
  }
}

__global__ __launch_bounds__(kVerifyThreads) void verify_kernel(VerifyKernelArgs a) {
  __shared__ VerifyShared s;
  const int b = blockIdx.x, tid = threadIdx.x;
  const std::size_t row0 = static_cast<std::size_t>(b) * a.nodes;
  const int count = a.node_counts != nullptr ? min(max(a.node_counts[b], 0), a.nodes) : a.nodes;
  const float* const target = a.target + b * a.target_batch_stride;
  const float* const draft = a.draft != nullptr ? a.draft + b * a.draft_batch_stride : nullptr;
  if (tid < kNodes) {
    int parent = -1, x = -1;
    double u = 0.0, p = 0.0, q = 0.0;
    if (tid < count) {
      parent = a.parents != nullptr ? a.parents[row0 + tid] : tid - 1;
      x = a.tokens[row0 + tid];
      u = static_cast<double>(a.uniforms[row0 + tid]);
      // Only nodes behind their parent, with a token of the vocabulary, can be
      // reached.
      if (parent < 0 || parent >= tid || x < 0 || x >= a.vocab) parent = -1;
      if (parent >= 0) {
        p = static_cast<double>(target[parent * a.target_node_stride + x]);
        if (draft != nullptr) q = static_cast<double>(draft[parent * a.draft_node_stride + x]);
      }
    }
    s.parent[tid] = parent;
    s.token[tid] = x;
    s.u[tid] = u;
    s.p[tid] = p;
    s.q[tid] = q;
    s.path[tid] = -1;
  }
  __syncthreads();
  int at = 0, number = count > 0 ? 1 : 0, rejected = 0;
  double mass = 1.0;
  Residual r{target, draft, s.totals, s.gone, 0};
  if (tid == 0 && count > 0) s.path[0] = 0;
  for (int c = 1; c < count; ++c) {
    if (s.parent[c] != at) continue;
    // The child's entry of the row that is left.
    double w = positive(s.p[c]);
    if (draft == nullptr) {
      for (int i = 0; i < rejected; ++i) w = s.gone[i] == s.token[c] ? 0.0 : w;
    } else {
      for (int i = 0; i < rejected; ++i) {
        w = positive(w - s.q[c]);
        if (s.totals[i] > 0.0) w /= s.totals[i];
      }
    }
    if (s.u[c] * (draft == nullptr ? mass : s.q[c]) < w) {
      at = c;
      if (tid == 0) s.path[number] = c;
      ++number;
      rejected = 0;
      mass = 1.0;
      r.p = target + at * a.target_node_stride;
      r.q = draft != nullptr ? draft + at * a.draft_node_stride : nullptr;
      r.rejected = 0;
      __syncthreads();  // every thread is done with the node's `gone` and `totals`
      continue;
    }
    mass -= w;
    if (tid == 0) s.gone[rejected] = s.token[c];
    r.rejected = ++rejected;
    if (draft != nullptr) {
      range_sums(r, true, 0, a.vocab, s);
      double total = 0.0;
      for (int i = 0; i < kVerifyWaves; ++i) total += s.part[i];
      if (tid == 0) s.totals[rejected - 1] = total;
    }
    __syncthreads();
  }
  int next = -1;
  if (count > 0) {
    const double bonus = static_cast<double>(a.bonus_uniforms[b]);
    next = pick(r, bonus, a.vocab, s);
    if (next < 0 && rejected > 0) {
      // Rounding left nothing of the row: its own probabilities stand.
      r.rejected = 0;
      next = pick(r, bonus, a.vocab, s);
    }
  }
  if (tid < a.nodes) a.path[row0 + tid] = s.path[tid];
  if (tid == 0) {
    a.accepted[b] = number;
    a.next_token[b] = next;
  }
}

}  // namespace

std::size_t verify_workspace_bytes(std::size_t, std::size_t, std::size_t) { return 256; }

hipError_t launch_verify(const VerifyArgs& a, hipStream_t stream) {
  if (a.batch == 0 || a.nodes == 0) return hipSuccess;
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
  k.nodes = static_cast<int>(a.nodes);
  k.vocab = static_cast<int>(a.vocab);
  verify_kernel<<<dim3(static_cast<unsigned>(a.batch)), kVerifyThreads, 0, stream>>>(k);
  return hipGetLastError();
}

}  // namespace helix::hip
