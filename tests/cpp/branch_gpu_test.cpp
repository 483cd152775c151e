// Several continuations of one prompt through the host API: state rows that fork, move and are cleared, tokens drawn from given numbers under
// options of their own, and the engine's loop over both.
#include <algorithm>
#include <cmath>

#include "rwkv_inference_engine.hpp"
#include "test_common.hpp"

using namespace rwkv7_server;

namespace {

constexpr int kVocab = 2048;

std::shared_ptr<ModelBackend> tiny(bool wkv32 = true) {
  static std::shared_ptr<ModelBackend> of[2];
  if (!of[wkv32]) of[wkv32] = std::make_shared<ModelBackend>("synthetic:tiny:w8:seed=3", wkv32);
  return of[wkv32];
}

std::shared_ptr<TrieTokenizer> tokenizer() {
  static std::shared_ptr<TrieTokenizer> tok = [] {
    auto t = std::make_shared<TrieTokenizer>();
    if (t->load(host_test::vocab_path()) != kTokenizerSuccess) throw std::runtime_error("vocab load failed");
    return t;
  }();
  return tok;
}

std::vector<int64_t> ramp(int n, int start) {
  std::vector<int64_t> v;
  for (int i = 0; i < n; ++i) v.push_back((start + 37 * i) % kVocab);
  return v;
}

// the bytes of every row of a state, tensor by tensor and plane by plane
std::vector<std::vector<uint8_t>> rows_of(const GenerationState& s, const rwkv7_fast_v4::ModelDims& d) {
  std::vector<std::vector<uint8_t>> out(s.batch_size);
  const auto add = [&](const void* p, std::size_t planes, std::size_t bytes) {
    std::vector<uint8_t> all(planes * s.batch_size * bytes);
    rwkv7_fast_v4::check_hip(rwkv_hip_memcpy_d2h(all.data(), p, all.size()), "test d2h");
    for (std::size_t l = 0; l < planes; ++l)
      for (int b = 0; b < s.batch_size; ++b) {
        const auto at = all.begin() + (l * s.batch_size + b) * bytes;
        out[b].insert(out[b].end(), at, at + bytes);
      }
  };
  add(s.shift.p, 2 * d.layers, 2 * d.channels);
  if (s.wkv32) add(s.wkv_state32.p, d.layers, std::size_t(4) * d.heads * 64 * 64);
  else add(s.wkv_state.p, d.layers, std::size_t(2) * d.heads * 64 * 64);
  add(s.elapsed.p, 1, 4);
  return out;
}

DeviceLogits make_logits(const std::vector<float>& host, int rows) {
  DeviceLogits l;
  l.rows = rows;
  l.vocab_size = int(host.size()) / rows;
  host_test::to_device(host, l.values);
  return l;
}

}  // namespace

HOST_TEST(state_rows_fork_move_and_are_cleared) {
  for (const bool wkv32 : {true, false}) {
    auto b = tiny(wkv32);
    const auto& d = b->dims();
    GenerationState s = b->create_state(3);
    DeviceLogits logits;
    b->forward_prefill({ramp(6, 1), ramp(6, 2), ramp(6, 3)}, s, logits);
    const auto before = rows_of(s, d);
    const std::vector<uint8_t> empty(before[0].size(), 0);
    CHECK(before[0] != before[1] && before[1] != before[2]);
    // to a wider batch: twice the same row, an empty one, one place left as it is
    GenerationState wide = b->create_state(5);
    b->copy_state_rows(s, {2, 2, -1, 0}, wide, {0, 4, 1, 3});
    const auto got = rows_of(wide, d);
    CHECK(got[0] == before[2] && got[4] == before[2] && got[1] == empty && got[3] == before[0] && got[2] == empty);
    CHECK(rows_of(s, d) == before);
    // inside a state: two change places, one is cleared
    b->copy_state_rows(s, {2, 0, -1}, s, {0, 2, 1});
    const auto moved = rows_of(s, d);
    CHECK(moved[0] == before[2] && moved[2] == before[0] && moved[1] == empty);
    // what copies go on with is what their original goes on with
    b->forward_decode({7, 8, 9, 10, 7}, wide, logits);
    const auto z = host_test::to_host<float>(logits.values);
    CHECK(std::equal(z.begin(), z.begin() + kVocab, z.begin() + 4 * kVocab));
    CHECK(rows_of(wide, d)[0] == rows_of(wide, d)[4]);
  }
}

HOST_TEST(state_rows_that_are_refused) {
  auto b = tiny();
  GenerationState s = b->create_state(3), t = b->create_state(2), none;
  CHECK_THROWS(b->copy_state_rows(s, {1}, t, {0, 1}), "as many state rows");
  CHECK_THROWS(b->copy_state_rows(s, {3}, t, {0}), "out of range");
  CHECK_THROWS(b->copy_state_rows(s, {-2}, t, {0}), "out of range");
  CHECK_THROWS(b->copy_state_rows(s, {1}, t, {2}), "out of range");
  CHECK_THROWS(b->copy_state_rows(s, {1, 0}, t, {1, 1}), "two state rows for one place");
  CHECK_THROWS(b->copy_state_rows(s, {1}, none, {0}), "non-empty");
  GenerationState half_state = tiny(false)->create_state(3);
  CHECK_THROWS(b->copy_state_rows(half_state, {1}, t, {0}), "precision mismatch");
  b->copy_state_rows(s, {}, t, {});
}

HOST_TEST(slices_move_inside_their_own_state) {
  auto b = tiny();
  const auto& d = b->dims();
  for (const int up : {0, 1}) {
    GenerationState s = b->create_state(5);
    DeviceLogits logits;
    b->forward_prefill({ramp(3, 1), ramp(3, 2), ramp(3, 3), ramp(3, 4), ramp(3, 5)}, s, logits);
    const auto before = rows_of(s, d);
    b->copy_state_slice(s, up ? 0 : 1, s, up ? 1 : 0, 4);
    const auto got = rows_of(s, d);
    for (int i = 0; i < 5; ++i) CHECK(got[i] == before[up ? std::max(i - 1, 0) : std::min(i + 1, 4)]);
  }
}

HOST_TEST(draws_known_answers) {
  const float inf = INFINITY;
  auto l = make_logits({1, 1, -inf, 0, 0, 3, 0, 0, -inf, 2, -inf, 2}, 3);
  DrawState state = make_draw_state(4, 3);
  DrawOptions greedy, two;
  greedy.temperature = 0.0;
  two.top_k = 2;
  DrawnTokens got = draw_tokens(l, {two, greedy, DrawOptions()}, {0.75f, 0.9f, 0.25f}, state);
  CHECK(got.tokens == (std::vector<int>{1, 1, 1}));
  CHECK_NEAR(got.logprobs[0], -std::log(2.0), 1e-7);
  CHECK_EQ(got.logprobs[1], 0.0f);
  CHECK_NEAR(got.logprobs[2], -std::log(2.0), 1e-7);
  // all from one row; penalties of the first call's tokens: 0.5, then times 0.5 plus 0.25
  DrawOptions pen;
  pen.alpha_presence = 0.5;
  pen.alpha_frequency = 0.25;
  pen.alpha_decay = 0.5;
  pen.top_k = 1;
  for (int call = 0; call < 2; ++call) CHECK(draw_tokens(l, {pen, pen, pen}, {0, 0, 0}, state, {1, 1, 1}).tokens == (std::vector<int>{1, 1, 1}));
  const std::vector<float> after = host_test::to_host<float>(state.penalties);
  CHECK((std::vector<float>(after.begin(), after.begin() + 4) == std::vector<float>{0, 0.5, 0, 0}));
  // rows of penalties move like rows of a state
  DrawState narrow = make_draw_state(4, 2);
  copy_draw_rows(state, {2, -1}, narrow, {1, 0});
  const std::vector<float> moved = host_test::to_host<float>(narrow.penalties);
  CHECK((std::vector<float>(moved.begin(), moved.begin() + 8) == std::vector<float>{0, 0, 0, 0, 0, 0.5, 0, 0}));
  auto nothing = make_logits({-inf, -inf, -inf, -inf}, 1);
  DrawState one = make_draw_state(4, 1, false);
  CHECK(draw_tokens(nothing, {DrawOptions()}, {0.5f}, one).tokens == std::vector<int>{-1});
}

HOST_TEST(draws_that_are_refused) {
  auto l = make_logits({1, 2, 3, 4, 5, 6, 7, 8}, 2);
  DrawState state = make_draw_state(4, 2), other = make_draw_state(8, 2), bare = make_draw_state(4, 2, false);
  const DrawOptions o;
  DrawOptions bad;
  bad.temperature = -1.0;
  CHECK_THROWS(draw_tokens(l, {o, o}, {0.5f, 0.5f}, other), "does not match sampler state");
  CHECK_THROWS(draw_tokens(l, {o}, {0.5f}, state), "does not match its options");
  CHECK_THROWS(draw_tokens(l, {o, o}, {0.5f}, state), "a random number for every row");
  CHECK_THROWS(draw_tokens(l, {o, o}, {0.5f, 0.5f}, state, {0}), "does not match logits rows");
  CHECK_THROWS(draw_tokens(l, {o, o}, {0.5f, 0.5f}, state, {0, 2}), "logits row out of range");
  CHECK_THROWS(draw_tokens(l, {o, bad}, {0.5f, 0.5f}, state), "negative or not a number");
  CHECK_THROWS(draw_tokens(l, {o, o}, {0.5f, 1.5f}, state), "outside 0 .. 1");
  CHECK_THROWS(copy_draw_rows(state, {0}, bare, {0}), "do not match");
  CHECK_THROWS(copy_draw_rows(state, {0}, other, {0}), "do not match");
}

HOST_TEST(a_greedy_branch_is_what_the_engine_generates) {
  InferenceEngine engine(tiny(), tokenizer(), "tiny");
  const std::string prompt = "User: hi\n\nAssistant:";
  GenerateOptions options;
  options.max_tokens = 12;
  options.stop_tokens = {0};
  options.top_p = 0.0;
  options.alpha_presence = options.alpha_frequency = 0.0;
  const std::string want = engine.batch_generate({prompt}, options)[0];
  InferenceEngine::BranchOptions branch;
  branch.max_tokens = 12;
  branch.stop_tokens = {0};
  branch.draw.temperature = 0.0;
  const auto one = engine.branch_generate(prompt, 1, branch);
  CHECK_EQ(one.size(), std::size_t(1));
  CHECK_EQ(one[0].text, want);
  for (const float p : one[0].logprobs) CHECK_EQ(p, 0.0f);
  const auto five = engine.branch_generate(prompt, 5, branch);
  for (const auto& b : five) CHECK(b.tokens == five[0].tokens);
  // no step, and a first step that is the last
  branch.max_tokens = 0;
  for (const auto& b : engine.branch_generate(prompt, 3, branch)) CHECK(b.tokens.empty() && b.text.empty() && !b.stopped);
  branch.max_tokens = 1;
  branch.stop_tokens.clear();
  for (const auto& b : engine.branch_generate(prompt, 3, branch)) CHECK(b.tokens == std::vector<int>(five[0].tokens.begin(), five[0].tokens.begin() + 1));
  branch.stop_tokens = {five[0].tokens[0]};
  branch.max_tokens = 9;
  for (const auto& b : engine.branch_generate(prompt, 3, branch)) CHECK(b.tokens.empty() && b.stopped);
}

// Every token of every branch, given the tokens in front of it, against a pass of its own at width 1: a state or penalty row that went to the
// wrong place would show.  Logits of other widths differ by steps of fp16, up to 16 halves of one at magnitudes below 8, on either side of the
// difference that a log probability is.
HOST_TEST(branches_go_on_from_their_own_states) {
  constexpr double kOff = 2.0 * 16.0 * 0.001953125;
  auto b = tiny();
  InferenceEngine engine(b, tokenizer(), "tiny");
  const std::string prompt = "User: name some numbers\n\nAssistant:";
  InferenceEngine::BranchOptions o;
  o.max_tokens = 14;
  o.stop_tokens.clear();
  for (int t = 0; t < kVocab; t += 9) o.stop_tokens.push_back(t);  // one token in nine ends a branch: the batch shrinks on the way
  o.draw.temperature = 0.7;
  o.draw.alpha_presence = 0.5;
  o.draw.alpha_frequency = 0.25;
  o.draw.alpha_decay = 0.9;
  o.seed = 11;
  const auto branches = engine.branch_generate(prompt, 12, o);
  int stopped = 0, longest = 0;
  double worst = 0.0;
  for (const auto& branch : branches) {
    stopped += branch.stopped;
    longest = std::max(longest, int(branch.tokens.size()));
    CHECK_EQ(branch.tokens.size(), branch.logprobs.size());
    CHECK(branch.stopped || int(branch.tokens.size()) == o.max_tokens);
    CHECK_EQ(branch.text, tokenizer()->decode(branch.tokens));
    GenerationState s = b->create_state(1);
    DeviceLogits logits;
    engine.prefill_prompt(prompt, s, logits);
    std::vector<double> penalty(kVocab, 0.0);
    for (std::size_t i = 0; i < branch.tokens.size(); ++i) {
      const auto z = host_test::to_host<float>(logits.values);
      double most = -INFINITY, sum = 0.0;
      for (int v = 0; v < kVocab; ++v) most = std::max(most, (z[v] - penalty[v]) / 0.7);
      for (int v = 0; v < kVocab; ++v) sum += std::exp((z[v] - penalty[v]) / 0.7 - most);
      const int token = branch.tokens[i];
      CHECK(std::find(o.stop_tokens.begin(), o.stop_tokens.end(), token) == o.stop_tokens.end());
      worst = std::max(worst, std::fabs((z[token] - penalty[token]) / 0.7 - most - std::log(sum) - branch.logprobs[i]));
      for (int v = 0; v < kVocab; ++v) penalty[v] = penalty[v] * 0.9 + (v != token ? 0.0 : penalty[v] == 0.0 ? 0.5 : 0.25);
      b->forward_decode({token}, s, logits);
    }
  }
  std::printf("     %d of 12 stopped, longest %d, largest difference %.4f\n", stopped, longest, worst);
  CHECK(stopped >= 4 && longest >= 6);
  CHECK(worst <= kOff / 0.7);
}

HOST_TEST(a_branch_belongs_to_its_seed_and_place) {
  InferenceEngine engine(tiny(), tokenizer(), "tiny");
  InferenceEngine::BranchOptions o;
  o.max_tokens = 6;
  o.stop_tokens.clear();
  o.draw.top_p = 0.95;
  o.draw.min_p = 0.01;
  o.seed = 5;
  const auto four = engine.branch_generate("User: hi", 4, o), again = engine.branch_generate("User: hi", 4, o);
  for (int i = 0; i < 4; ++i) CHECK(four[i].tokens == again[i].tokens && four[i].logprobs == again[i].logprobs);
  const auto nine = engine.branch_generate("User: hi", 9, o);
  for (int i = 0; i < 4; ++i) CHECK_EQ(nine[i].tokens[0], four[i].tokens[0]);  // (drawn from the same logits)
  o.seed = 6;
  const auto other = engine.branch_generate("User: hi", 4, o);
  int same = 0;
  for (int i = 0; i < 4; ++i) same += other[i].tokens == four[i].tokens;
  CHECK(same < 4);
}

// Stop tokens that the model does not have are never drawn, and no branch that has ended is fed one
HOST_TEST(stop_tokens_outside_the_vocabulary) {
  InferenceEngine engine(tiny(), tokenizer(), "tiny");
  InferenceEngine::BranchOptions o;
  o.max_tokens = 10;
  o.seed = 3;
  o.stop_tokens.clear();
  for (int t = 0; t < kVocab; t += 9) o.stop_tokens.push_back(t);
  const auto want = engine.branch_generate("User: hi", 9, o);
  int stopped = 0;
  for (const auto& b : want) stopped += b.stopped;
  CHECK(stopped > 0 && stopped < 9);
  for (const int64_t outside : {int64_t{kVocab}, int64_t{70000}, int64_t{-1}}) {
    o.stop_tokens.insert(o.stop_tokens.begin(), outside);
    const auto got = engine.branch_generate("User: hi", 9, o);
    for (int i = 0; i < 9; ++i) CHECK(got[i].tokens == want[i].tokens && got[i].logprobs == want[i].logprobs && got[i].stopped == want[i].stopped);
  }
}

int main(int argc, char** argv) { return host_test::run_all(argc, argv, true); }
