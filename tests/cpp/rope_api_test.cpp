// Rotation with append of include/helix_paged.hpp (DecodeBatch::rope_append_layer),
// one-token and chunk steps, against sums in 64 bits.  Built by tests/cpp/Makefile;
// run by tests/test_cpp_rope_api.py.  Without a GPU the case reports SKIPPED.
#include "helix_paged.hpp"
#include "mini_test.hpp"

#include <array>
#include <cmath>
#include <cstdint>
#include <vector>

namespace {

using namespace helix_amd;
using namespace helix_amd::kv_cache;
using Stream = helix_amd::hip::Stream;

struct RopeAppendTest {
  void SetUp() {
    if (!helix_amd::hip::runtime_available()) SKIP("requires a visible AMD GPU");
    helix_amd::hip::set_device(0);
  }
};

const Device kGpu = Device::gpu(0);
constexpr std::size_t L = 2, H = 2, HQ = 4, D = 128, P = 16, B = 2, T = 5, R = 64;

Tensor ramp(Shape shape, float from) {
  std::vector<float> v(shape_numel(shape));
  for (std::size_t i = 0; i < v.size(); ++i) v[i] = from + 0.001F * static_cast<float>(i % 997);
  return Tensor::from_values(std::move(shape), v);
}

// Rows [B, heads, tokens, D] turned, sequence b's first one at position starts[b].
std::vector<double> turned(const Tensor& rows, std::size_t heads, std::size_t tokens,
                           const std::array<std::size_t, B>& starts, helix_rope_layout layout) {
  const float* const x = rows.data_as<float>();
  std::vector<double> y(x, x + rows.numel());
  for (std::size_t b = 0; b < B; ++b)
    for (std::size_t h = 0; h < heads; ++h)
      for (std::size_t t = 0; t < tokens; ++t)
        for (std::size_t i = 0; i < R / 2; ++i) {
          const std::size_t at = ((b * heads + h) * tokens + t) * D;
          const std::size_t one = at + (layout == HELIX_ROPE_PAIRS ? 2 * i : i);
          const std::size_t two = layout == HELIX_ROPE_PAIRS ? one + 1 : one + R / 2;
          const double angle = static_cast<double>(starts[b] + t) *
                               std::pow(10000.0, -2.0 * static_cast<double>(i) / R);
          y[one] = x[one] * std::cos(angle) - x[two] * std::sin(angle);
          y[two] = x[one] * std::sin(angle) + x[two] * std::cos(angle);
        }
  return y;
}

// Inputs below 1.6: two products and a sum, and tables, rounded to 2^-24 each, are
// below 1e-6 together.
void near(const Tensor& got, const std::vector<double>& want) {
  const Tensor host = got.to(Device::cpu());
  for (std::size_t i = 0; i < want.size(); ++i) EXPECT_NEAR(host.data_as<float>()[i], want[i], 1e-6);
}

TEST_F(RopeAppendTest, StepsRotateAndAppend) {
  HipPagedKvCache cache(PagedKvCacheConfig{L, H, D, P, 16});
  Stream stream;
  const std::array<HipPagedSequenceHandle, B> seqs{cache.create_sequence(),
                                                   cache.create_sequence()};
  const std::vector<Tensor> history(L, ramp({H, 7, D}, -0.5F).to(kGpu));
  cache.append_layer_major(seqs[1], history, history, stream);
  DecodeBatch batch(cache, seqs, HQ, 64);
  Tensor cosine = Tensor::empty({64, R / 2}, DType::kFloat32, kGpu);
  Tensor sine = Tensor::empty({64, R / 2}, DType::kFloat32, kGpu);
  EXPECT_EQ(helix_rope_tables(cosine.data<float>(), sine.data<float>(), 64, 0, R, 10000.0,
                              HELIX_ROPE_SCALE_NONE, 1.0, 0.0, 1.0, 32.0, 1.0, stream.native()),
            0);

  std::array<std::size_t, B> starts{0, 7};
  for (const std::size_t tokens : {std::size_t{1}, T}) {
    const bool chunk = tokens != 1;
    const auto layout = chunk ? HELIX_ROPE_HALVES : HELIX_ROPE_PAIRS;
    const auto shape = [&](std::size_t heads) {
      const std::int64_t n = static_cast<std::int64_t>(heads);
      return chunk ? Shape{B, n, T, D} : Shape{B, n, D};
    };
    chunk ? batch.prepare_chunk(T, stream) : batch.prepare(stream);
    const Tensor q_host = ramp(shape(HQ), 0.1F), k_host = ramp(shape(H), 0.2F);
    const Tensor v_host = ramp(shape(H), 0.3F);
    const Tensor q = q_host.to(kGpu), v = v_host.to(kGpu);
    Tensor q_out = Tensor::empty(shape(HQ), DType::kFloat32, kGpu);
    Tensor k = k_host.to(kGpu);  // (rotated in place)
    for (std::size_t l = 0; l < L; ++l) {
      Tensor layer_key = l == 0 ? k_host.to(kGpu) : k;
      batch.rope_append_layer(l, q, layer_key, v, q_out, layer_key, cosine, sine, layout, stream);
      if (l == 0) stream.synchronize();
    }
    EXPECT_THROW(batch.rope_append_layer(0, k, k, v, q_out, k, cosine, sine, layout, stream), Error);
    EXPECT_THROW(batch.rope_append_layer(0, q, k, v, q_out, k, cosine, q, layout, stream), Error);
    stream.synchronize();
    near(q_out, turned(q_host, HQ, tokens, starts, layout));
    const std::vector<double> keys = turned(k_host, H, tokens, starts, layout);
    near(k, keys);

    // The pages have the same rows, and the values bit by bit.
    for (std::size_t b = 0; b < B; ++b) {
      const std::size_t all = starts[b] + tokens;
      EXPECT_EQ(cache.length(seqs[b]), all);
      const Shape out{static_cast<std::int64_t>(H), static_cast<std::int64_t>(all), D};
      Tensor k_page = Tensor::empty(out, DType::kFloat32, kGpu);
      Tensor v_page = Tensor::empty(out, DType::kFloat32, kGpu);
      cache.copy_layer_out(seqs[b], 1, k_page, v_page, stream);
      stream.synchronize();
      const Tensor kp = k_page.to(Device::cpu()), vp = v_page.to(Device::cpu());
      for (std::size_t h = 0; h < H; ++h)
        for (std::size_t t = 0; t < tokens; ++t)
          for (std::size_t d = 0; d < D; ++d) {
            const std::size_t row = ((b * H + h) * tokens + t) * D + d;
            const std::size_t page = (h * all + starts[b] + t) * D + d;
            EXPECT_NEAR(kp.data_as<float>()[page], keys[row], 1e-6);
            EXPECT_EQ(vp.data_as<float>()[page], v_host.data_as<float>()[row]);
          }
      starts[b] = all;
    }
  }
}

}  // namespace

int main(int argc, char** argv) {
  return mini_test::run_all(argc > 1 ? argv[1] : nullptr);
}
