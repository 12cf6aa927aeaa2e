// The tree step of include/helix_paged.hpp: DecodeBatch::prepare_tree,
// tree_layer, commit_path and accept_tree, and truncate_sequence, on a small
// batch whose results are known.  Built by tests/cpp/Makefile; run by
// tests/test_cpp_tree_api.py.  Without a GPU the cases report SKIPPED.
#include "helix_paged.hpp"
#include "mini_test.hpp"

#include <array>
#include <cstdint>
#include <vector>

namespace {

using namespace helix_amd;
using namespace helix_amd::kv_cache;
using Stream = helix_amd::hip::Stream;

struct TreeStepTest {
  void SetUp() {
    if (!helix_amd::hip::runtime_available()) SKIP("requires a visible AMD GPU");
    helix_amd::hip::set_device(0);
  }
};

const Device kGpu = Device::gpu(0);
constexpr std::size_t L = 2, H = 2, HQ = 4, D = 128, P = 16, B = 2, T = 3, V = 7;

Tensor ramp(Shape shape, float from) {
  std::vector<float> v(shape_numel(shape));
  for (std::size_t i = 0; i < v.size(); ++i) v[i] = from + 0.001F * static_cast<float>(i % 997);
  return Tensor::from_values(std::move(shape), v);
}

Tensor ints(Shape shape, const std::vector<std::int32_t>& v) {
  Tensor t = Tensor::empty(std::move(shape), DType::kInt32, Device::cpu());
  std::copy(v.begin(), v.end(), t.data<std::int32_t>());
  return t.to(kGpu);
}

std::vector<std::int32_t> host_ints(const Tensor& t) {
  const Tensor h = t.to(Device::cpu());
  return {h.data_as<std::int32_t>(), h.data_as<std::int32_t>() + h.numel()};
}

TEST_F(TreeStepTest, AStepKeepsWhatTheTargetAccepts) {
  HipPagedKvCache cache(PagedKvCacheConfig{L, H, D, P, 16});
  Stream stream;
  const std::array<HipPagedSequenceHandle, B> seqs{cache.create_sequence(),
                                                   cache.create_sequence()};
  const std::vector<Tensor> history(L, ramp({H, 5, D}, -0.5F).to(kGpu));
  cache.append_layer_major(seqs[1], history, history, stream);
  DecodeBatch batch(cache, seqs, HQ, 64);

  batch.prepare_tree(T, stream);
  const Tensor q = ramp({B, HQ, T, D}, 0.1F).to(kGpu);
  const Tensor key_host = ramp({L, B, H, T, D}, 0.2F), value_host = ramp({L, B, H, T, D}, 0.3F);
  const Tensor keys = key_host.to(kGpu), values = value_host.to(kGpu);
  const Tensor layer_key = ramp({B, H, T, D}, 0.2F).to(kGpu);
  const Tensor layer_value_host = ramp({B, H, T, D}, 0.3F);
  const Tensor layer_value = layer_value_host.to(kGpu);
  // Nodes 1 and 2 are children of node 0.
  const Tensor parents = ints({B, T}, {-1, 0, 0, -1, 0, 0});
  Tensor out = Tensor::empty({B, HQ, T, D}, DType::kFloat32, kGpu);
  batch.tree_layer(0, q, layer_key, layer_value, &parents, nullptr, out, stream);
  EXPECT_THROW(batch.tree_layer(0, q, layer_key, layer_value, &out, nullptr, out, stream), Error);
  stream.synchronize();
  // A root without history sees itself alone.
  const Tensor seen = out.to(Device::cpu());
  for (std::size_t h = 0; h < HQ; ++h) {
    for (std::size_t d = 0; d < D; ++d) {
      EXPECT_NEAR(seen.data_as<float>()[h * T * D + d],
                  layer_value_host.data_as<float>()[h / (HQ / H) * T * D + d], 1e-6F);
    }
  }

  // The target is certain: token 4 behind the root, 6 behind node 2.  Of the
  // first sequence's drafts node 2 has it, of the second's none.
  std::vector<float> p(B * T * V, 0.0F);
  for (std::size_t b = 0; b < B; ++b) {
    p[(b * T + 0) * V + 4] = p[(b * T + 1) * V + 5] = p[(b * T + 2) * V + 6] = 1.0F;
  }
  const Tensor target = Tensor::from_values({B, T, V}, p).to(kGpu);
  const Tensor tokens = ints({B, T}, {0, 1, 4, 0, 1, 2});
  const Tensor uniforms = Tensor::from_values({B, T}, std::vector<float>(B * T, 0.5F)).to(kGpu);
  const Tensor bonus = Tensor::from_values({B}, std::vector<float>(B, 0.5F)).to(kGpu);
  Tensor path = ints({B, T}, std::vector<std::int32_t>(B * T, 9));
  Tensor accepted = ints({B}, {9, 9}), next = ints({B}, {9, 9});
  batch.accept_tree(target, nullptr, tokens, &parents, nullptr, uniforms, bonus, keys, values,
                    path, accepted, next, stream);
  EXPECT_TRUE((host_ints(path) == std::vector<std::int32_t>{0, 2, -1, 0, -1, -1}));
  EXPECT_TRUE((host_ints(accepted) == std::vector<std::int32_t>{2, 1}));
  EXPECT_TRUE((host_ints(next) == std::vector<std::int32_t>{6, 4}));
  EXPECT_EQ(cache.length(seqs[0]), 2U);
  EXPECT_EQ(cache.length(seqs[1]), 6U);

  // The accepted rows, bit by bit.
  Tensor k_out = Tensor::empty({H, 2, D}, DType::kFloat32, kGpu);
  Tensor v_out = Tensor::empty({H, 2, D}, DType::kFloat32, kGpu);
  cache.copy_layer_out(seqs[0], 1, k_out, v_out, stream);
  const Tensor got = v_out.to(Device::cpu());
  const float* const rows = value_host.data_as<float>() + B * H * T * D;  // layer 1
  for (std::size_t h = 0; h < H; ++h) {
    for (std::size_t i = 0; i < 2; ++i) {
      for (std::size_t d = 0; d < D; ++d) {
        EXPECT_EQ(got.data_as<float>()[(h * 2 + i) * D + d], rows[(h * T + 2 * i) * D + d]);
      }
    }
  }

  // commit_path by itself, then back again.
  batch.prepare_tree(T, stream);
  const Tensor chosen = ints({B, T}, {0, 1, 2, 0, -1, -1}), numbers = ints({B}, {3, 0});
  EXPECT_THROW(batch.commit_path(layer_key, values, chosen, numbers, stream), Error);
  batch.commit_path(keys, values, chosen, numbers, stream);
  EXPECT_EQ(cache.length(seqs[0]), 5U);
  EXPECT_EQ(cache.length(seqs[1]), 6U);
  cache.truncate_sequence(seqs[0], 1);
  EXPECT_EQ(cache.length(seqs[0]), 1U);
  EXPECT_THROW(cache.truncate_sequence(seqs[0], 2), Error);
}

}  // namespace

int main(int argc, char** argv) {
  return mini_test::run_all(argc > 1 ? argv[1] : nullptr);
}
