// Rows of draw states that are refused, and numbers of continuations, before a device is touched.
#include <numeric>

#include "rwkv_inference_engine.hpp"
#include "test_common.hpp"

using namespace rwkv7_server;

namespace {

// (of a state without penalties nothing moves, but what is asked for is looked at all the same)
DrawState rows_of(int batch_size) {
  DrawState s;
  s.batch_size = batch_size;
  s.vocab_size = 100;
  return s;
}

std::vector<int> numbers(int n, int first = 0) {
  std::vector<int> v(n);
  std::iota(v.begin(), v.end(), first);
  return v;
}

// counts what is asked of it
class Counting final : public IModelBackend {
 public:
  GenerationState create_state(int) const override {
    ++calls;
    throw std::runtime_error("a state was created");
  }
  void copy_state_slice(const GenerationState&, int, GenerationState&, int, int) const override {}
  void forward_prefill(const std::vector<std::vector<int64_t>>&, GenerationState&, DeviceLogits&) const override {}
  void forward_decode(const std::vector<int64_t>&, GenerationState&, DeviceLogits&) const override {}
  void copy_logits_slice(const DeviceLogits&, int, DeviceLogits&, int, int) const override {}
  PrefillCapacity query_prefill_capacity(int) const override { return {}; }
  int vocab_size() const override { return 100; }
  const std::string& model_path() const override { return name_; }
  const std::string& model_name() const override { return name_; }
  mutable int calls = 0;

 private:
  std::string name_ = "counting";
};

}  // namespace

HOST_TEST(draw_rows_that_are_refused) {
  DrawState s = rows_of(3), t = rows_of(2), wide = rows_of(2000);
  CHECK_THROWS(copy_draw_rows(s, {1}, t, {0, 1}), "as many draw rows");
  CHECK_THROWS(copy_draw_rows(s, {3}, t, {0}), "draw row out of range");
  CHECK_THROWS(copy_draw_rows(s, {-2}, t, {0}), "draw row out of range");
  CHECK_THROWS(copy_draw_rows(s, {1}, t, {2}), "draw row out of range");
  CHECK_THROWS(copy_draw_rows(s, {1}, t, {-1}), "draw row out of range");
  CHECK_THROWS(copy_draw_rows(s, {1, 0}, t, {1, 1}), "two draw rows for one place");
  CHECK_THROWS(copy_draw_rows(wide, numbers(513), wide, numbers(513)), "more than 512 rows");
  copy_draw_rows(s, {2, -1}, t, {0, 1});
  copy_draw_rows(s, {}, t, {});
  // behind the rows of the first launch
  DrawState other = rows_of(2000);
  std::vector<int> to = numbers(1000);
  to[900] = 5;
  CHECK_THROWS(copy_draw_rows(wide, numbers(1000), other, to), "two draw rows for one place");
  to[900] = 2000;
  CHECK_THROWS(copy_draw_rows(wide, numbers(1000), other, to), "draw row out of range");
  DrawState many = rows_of(65535);
  CHECK_THROWS(copy_draw_rows(s, {0}, many, {0}), "more than 65534 rows");
  CHECK_THROWS(copy_draw_rows(many, {0}, s, {0}), "more than 65534 rows");
}

HOST_TEST(numbers_of_continuations_that_are_refused) {
  auto backend = std::make_shared<Counting>();
  InferenceEngine engine(backend, std::make_shared<TrieTokenizer>(), "counting");
  for (const int n : {0, -1, 65535, 2147483647}) CHECK_THROWS(engine.branch_generate("x", n, {}), "number of continuations must");
  CHECK_EQ(backend->calls, 0);
  CHECK_THROWS(engine.branch_generate("x", 65534, {}), "a state was created");
}

int main(int argc, char** argv) { return host_test::run_all(argc, argv, false); }
