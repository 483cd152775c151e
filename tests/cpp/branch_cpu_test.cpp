// What several continuations of a prompt need of the host side: moving state rows over a backend that only has slices, and their random
// numbers.  No GPU.
#include <algorithm>
#include <set>

#include "rwkv_inference_engine.hpp"
#include "test_common.hpp"

using namespace rwkv7_server;

namespace {

// a backend that writes down its slices
class SliceBackend final : public IModelBackend {
 public:
  struct Slice {
    int from, to, count;
    bool operator==(const Slice& o) const { return from == o.from && to == o.to && count == o.count; }
  };
  GenerationState create_state(int batch_size) const override {
    GenerationState s;
    s.batch_size = batch_size;
    return s;
  }
  void copy_state_slice(const GenerationState&, int from, GenerationState&, int to, int count) const override { slices.push_back({from, to, count}); }
  void forward_prefill(const std::vector<std::vector<int64_t>>&, GenerationState&, DeviceLogits&) const override {}
  void forward_decode(const std::vector<int64_t>&, GenerationState&, DeviceLogits&) const override {}
  void copy_logits_slice(const DeviceLogits&, int, DeviceLogits&, int, int) const override {}
  PrefillCapacity query_prefill_capacity(int) const override { return {}; }
  int vocab_size() const override { return 100; }
  const std::string& model_path() const override { return name_; }
  const std::string& model_name() const override { return name_; }
  mutable std::vector<Slice> slices;

 private:
  std::string name_ = "slices";
};

}  // namespace

HOST_TEST(backends_with_slices_move_runs_of_rows) {
  SliceBackend b;
  GenerationState src = b.create_state(9), dst = b.create_state(6);
  b.copy_state_rows(src, {2, 3, 4, 7, 0, 0}, dst, {0, 1, 2, 3, 4, 5});
  CHECK(b.slices == (std::vector<SliceBackend::Slice>{{2, 0, 3}, {7, 3, 1}, {0, 4, 1}, {0, 5, 1}}));
  b.slices.clear();
  b.copy_state_rows(src, {}, dst, {});
  CHECK(b.slices.empty());
  CHECK_THROWS(b.copy_state_rows(src, {1}, dst, {}), "as many state rows");
  CHECK_THROWS(b.copy_state_rows(src, {-1}, dst, {0}), "does not clear");
  CHECK_THROWS(b.copy_state_rows(src, {1}, src, {0}), "inside a state");
}

HOST_TEST(numbers_depend_on_their_place_alone) {
  std::set<float> seen;
  double sum = 0.0, square = 0.0;
  int low = 0;
  constexpr int kSequences = 100, kSteps = 200;
  for (int i = 0; i < kSequences; ++i)
    for (int t = 0; t < kSteps; ++t) {
      const float u = uniform_of(42, i, t);
      CHECK(u >= 0.0f && u < 1.0f);
      CHECK_EQ(u, uniform_of(42, i, t));
      CHECK_EQ(u * 16777216.0f, std::floor(u * 16777216.0f));
      seen.insert(u);
      sum += u;
      square += u * u;
      low += u < 0.25f;
    }
  constexpr double n = kSequences * kSteps;
  // five standard deviations of the average of n uniform numbers, of their squares and of a count
  CHECK_NEAR(sum / n, 0.5, 5.0 * std::sqrt(1.0 / 12.0 / n));
  CHECK_NEAR(square / n, 1.0 / 3.0, 5.0 * std::sqrt(4.0 / 45.0 / n));
  CHECK_NEAR(low / n, 0.25, 5.0 * std::sqrt(0.25 * 0.75 / n));
  CHECK(seen.size() > n - 60);  // (of 2^24 places: twelve pairs share one on average)
  CHECK(uniform_of(1, 2, 3) != uniform_of(1, 3, 2));
  CHECK(uniform_of(1, 2, 3) != uniform_of(2, 2, 3));
}

HOST_TEST(what_is_refused_before_a_device_is_touched) {
  CHECK_THROWS(make_draw_state(0, 1), "invalid sampler vocab size");
  CHECK_THROWS(make_draw_state(100, 0), "invalid sampler batch size");
  CHECK_THROWS(make_draw_state(2000000, 1), "bad arguments");
  DrawState none;
  DeviceLogits logits;
  CHECK_THROWS(draw_tokens(logits, {}, {}, none), "at least one logits row");
  logits.rows = 2;
  logits.vocab_size = 100;
  CHECK_THROWS(draw_tokens(logits, {}, {}, none), "empty device logits");
  auto backend = std::make_shared<SliceBackend>();
  InferenceEngine engine(backend, std::make_shared<TrieTokenizer>(), "slices");
  CHECK_THROWS(engine.branch_generate("x", 0, {}), "must be positive");
}

int main(int argc, char** argv) { return host_test::run_all(argc, argv, false); }
