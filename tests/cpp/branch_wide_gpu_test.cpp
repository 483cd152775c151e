// States of more rows than one launch of rwkv_hip_copy_rows numbers (65534): slices and rows of them move all the same.
#include <algorithm>

#include "rwkv_server_backend.hpp"
#include "test_common.hpp"

using namespace rwkv7_server;

namespace {

constexpr int kWide = 65600;

std::shared_ptr<ModelBackend> tiny() {
  static auto b = std::make_shared<ModelBackend>("synthetic:tiny:w8:seed=3", false);
  return b;
}

// the bytes of one row of a state, tensor by tensor and plane by plane
std::vector<uint8_t> row_of(const GenerationState& s, int row) {
  const auto& d = tiny()->dims();
  std::vector<uint8_t> out;
  const auto add = [&](const void* p, std::size_t planes, std::size_t bytes) {
    for (std::size_t l = 0; l < planes; ++l) {
      out.resize(out.size() + bytes);
      rwkv7_fast_v4::check_hip(rwkv_hip_memcpy_d2h(out.data() + out.size() - bytes, static_cast<const char*>(p) + (l * s.batch_size + row) * bytes, bytes),
                               "test d2h");
    }
  };
  add(s.shift.p, 2 * d.layers, 2 * d.channels);
  add(s.wkv_state.p, d.layers, std::size_t(2) * d.heads * 64 * 64);
  add(s.elapsed.p, 1, 4);
  return out;
}

// three rows that differ
GenerationState three() {
  GenerationState s = tiny()->create_state(3);
  DeviceLogits logits;
  tiny()->forward_prefill({{1, 38, 75}, {2, 39, 76}, {3, 40, 77}}, s, logits);
  return s;
}

}  // namespace

HOST_TEST(slices_of_a_wide_state) {
  auto b = tiny();
  GenerationState s = three(), wide = b->create_state(kWide), back = b->create_state(5);
  b->copy_state_slice(s, 0, wide, 65560, 3);
  for (int i = 0; i < 3; ++i) CHECK(row_of(wide, 65560 + i) == row_of(s, i));
  const auto empty = row_of(back, 0);
  CHECK(row_of(wide, 65559) == empty && row_of(wide, 65563) == empty);
  b->copy_state_slice(wide, 65561, back, 2, 2);
  CHECK(row_of(back, 2) == row_of(s, 1) && row_of(back, 3) == row_of(s, 2) && row_of(back, 1) == empty && row_of(back, 4) == empty);
  // one place on, and back, inside the state
  b->copy_state_slice(wide, 65559, wide, 65560, 4);
  for (int i = 0; i < 3; ++i) CHECK(row_of(wide, 65561 + i) == row_of(s, i));
  CHECK(row_of(wide, 65560) == empty);
  b->copy_state_slice(wide, 65560, wide, 65559, 4);
  for (int i = 0; i < 3; ++i) CHECK(row_of(wide, 65560 + i) == row_of(s, i));
  CHECK(row_of(wide, 65563) == row_of(s, 2));
}

HOST_TEST(rows_of_a_wide_state) {
  auto b = tiny();
  GenerationState s = three(), wide = b->create_state(kWide), back = b->create_state(4);
  const auto empty = row_of(back, 0);
  b->copy_state_rows(s, {2, 0, 1, 1}, wide, {65599, 65540, 0, 65541});
  CHECK(row_of(wide, 65599) == row_of(s, 2) && row_of(wide, 65540) == row_of(s, 0) && row_of(wide, 0) == row_of(s, 1) &&
        row_of(wide, 65541) == row_of(s, 1) && row_of(wide, 65542) == empty);
  // inside the state: two change places, one forks, one is cleared
  b->copy_state_rows(wide, {65540, 65599, 65599, -1}, wide, {65599, 65540, 7, 65541});
  CHECK(row_of(wide, 65599) == row_of(s, 0) && row_of(wide, 65540) == row_of(s, 2) && row_of(wide, 7) == row_of(s, 2) && row_of(wide, 65541) == empty);
  b->copy_state_rows(wide, {0, 1}, back, {2, 3});
  b->copy_state_rows(wide, {65599, 7, -1}, back, {3, 0, 2});
  CHECK(row_of(back, 3) == row_of(s, 0) && row_of(back, 0) == row_of(s, 2) && row_of(back, 2) == empty);
  CHECK_THROWS(b->copy_state_rows(wide, {kWide}, back, {0}), "out of range");
  CHECK_THROWS(b->copy_state_rows(wide, {0, 1}, back, {2, 2}), "two state rows for one place");
  CHECK_THROWS(b->copy_state_rows(back, {0}, wide, {kWide}), "out of range");
}

int main(int argc, char** argv) { return host_test::run_all(argc, argv, true); }
