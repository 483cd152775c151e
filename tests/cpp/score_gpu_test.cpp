// Log probabilities through the host API: beside the sampler, at every position of a backend's call, and of whole texts.
#include <algorithm>
#include <cmath>

#include "rwkv_inference_engine.hpp"
#include "scripted_backend.hpp"

using namespace rwkv7_server;

namespace {

std::shared_ptr<ModelBackend> tiny() {
  static auto backend = std::make_shared<ModelBackend>("synthetic:tiny:w8:seed=3", true);
  return backend;
}

std::vector<int64_t> ramp(int n, int start) {
  std::vector<int64_t> v;
  for (int i = 0; i < n; ++i) v.push_back((start + 37 * i) % 2048);
  return v;
}

DeviceLogits make_logits(const std::vector<float>& host, int rows) {
  DeviceLogits l;
  l.rows = rows;
  l.vocab_size = int(host.size()) / rows;
  host_test::to_device(host, l.values);
  return l;
}

double log_softmax(const std::vector<float>& z, int64_t t) {
  double m = z[0], s = 0;
  for (float v : z) m = std::max(m, double(v));
  for (float v : z) s += std::exp(v - m);
  return z[t] - m - std::log(s);
}

}  // namespace

HOST_TEST(token_logprobs_known_answers) {
  const float inf = INFINITY;
  // two equal ones; one sure; a masked row with two left
  auto l = make_logits({1, 1, -inf, -inf, 0, 100, 0, 0, -inf, 2, -inf, 2}, 3);
  const TokenLogprobs p = token_logprobs(l, {1, 1, -1}, 3);
  CHECK_EQ(p.rows, 3);
  CHECK_NEAR(p.logprob[0], -std::log(2.0), 1e-6);
  CHECK_NEAR(p.entropy[0], std::log(2.0), 1e-6);
  CHECK_NEAR(p.logprob[1], 0.0, 1e-6);
  CHECK_NEAR(p.entropy[1], 0.0, 1e-6);
  CHECK_EQ(p.logprob[2], 0.0f);
  CHECK(p.rank == (std::vector<int>{1, 0, -1}));
  CHECK(p.top_ids == (std::vector<int>{0, 1, -1, 1, 0, 2, 1, 3, -1}));
  CHECK_NEAR(p.top_logprobs[6], -std::log(2.0), 1e-6);
  CHECK(std::isinf(p.top_logprobs[2]) && p.top_logprobs[2] < 0);
}

HOST_TEST(token_logprobs_errors) {
  auto l = make_logits({1, 2, 3, 4}, 1);
  CHECK_THROWS(token_logprobs(l, {0, 1}), "a token per logits row");
  CHECK_THROWS(token_logprobs(l, {4}), "token id out of range");
  CHECK_THROWS(token_logprobs(l, {-2}), "token id out of range");
  CHECK_THROWS(token_logprobs(l, {0}, 65), "top_n");
  CHECK_THROWS(token_logprobs(l, {0}, -1), "top_n");
  DeviceLogits empty;
  empty.rows = 1;
  CHECK_THROWS(token_logprobs(empty, {0}), "empty device logits");
}

HOST_TEST(sampled_token_has_the_log_probability_of_its_logits) {
  auto b = tiny();
  GenerationState s = b->create_state(2);
  DeviceLogits l;
  b->forward_prefill({ramp(9, 1), ramp(9, 2)}, s, l);
  auto penalties = make_sampler_penalties(b->vocab_size(), 2, 7);
  const std::vector<int> tokens = sample_batch_repetition_temperature_topk_topp(l, penalties, GenerateOptions{});
  const TokenLogprobs p = token_logprobs(l, tokens, 5);
  const auto z = host_test::to_host<float>(l.values);
  for (int r = 0; r < 2; ++r) {
    const std::vector<float> row(z.begin() + r * 2048, z.begin() + (r + 1) * 2048);
    CHECK_NEAR(p.logprob[r], log_softmax(row, tokens[r]), 1e-4);
    CHECK_EQ(p.top_ids[r * 5], int(std::max_element(row.begin(), row.end()) - row.begin()));
  }
}

// The logits of position i are those of a forward call that ends there; fp16 activations: cosine bars elsewhere, here a few hundredths.
HOST_TEST(backend_scores_every_position) {
  auto b = tiny();
  const int T = 11;
  const std::vector<int64_t> text = ramp(T + 1, 5), other = ramp(T + 1, 900);
  std::vector<std::vector<int64_t>> tokens = {{text.begin(), text.end() - 1}, {other.begin(), other.end() - 1}};
  std::vector<std::vector<int64_t>> targets = {{text.begin() + 1, text.end()}, {other.begin() + 1, other.end()}};
  targets[1][3] = -1;
  for (const bool int8 : {false, true}) {
    GenerationState s = b->create_state(2), step = b->create_state(2);
    ScoreOptions o;
    o.top_n = 2;
    o.int8_head = int8;
    const TokenLogprobs p = b->score(tokens, targets, s, o);
    CHECK_EQ(p.rows, 2 * T);
    DeviceLogits l;
    for (int t = 0; t < T; ++t) {
      b->forward_decode({tokens[0][t], tokens[1][t]}, step, l);
      const auto z = host_test::to_host<float>(l.values);
      for (int r = 0; r < 2; ++r) {
        const std::vector<float> row(z.begin() + r * 2048, z.begin() + (r + 1) * 2048);
        const double want = targets[r][t] < 0 ? 0.0 : log_softmax(row, targets[r][t]);
        CHECK_NEAR(p.logprob[r * T + t], want, 0.05);
        CHECK(p.top_logprobs[(r * T + t) * 2] >= p.top_logprobs[(r * T + t) * 2 + 1]);
        CHECK_NEAR(p.top_logprobs[(r * T + t) * 2], log_softmax(row, p.top_ids[(r * T + t) * 2]), 0.05);
      }
    }
    CHECK(host_test::to_host<int>(s.elapsed) == (std::vector<int>{T, T}));
  }
}

HOST_TEST(backend_score_errors) {
  auto b = tiny();
  GenerationState s = b->create_state(1);
  CHECK_THROWS(b->score({}, {}, s, {}), "token_batches must not be empty");
  CHECK_THROWS(b->score({{1, 2}, {3, 4}}, {{1, 2}, {3, 4}}, s, {}), "state batch size mismatch");
  CHECK_THROWS(b->score({{1, 2}}, {{1}}, s, {}), "target batches do not match");
  CHECK_THROWS(b->score({{1, 2}}, {}, s, {}), "target batches do not match");
  CHECK_THROWS(b->score({{1, 2}}, {{1, 2048}}, s, {}), "target id out of range");
  CHECK_THROWS(b->score({{1, 2}}, {{1, -2}}, s, {}), "target id out of range");
  CHECK_THROWS(b->score({{1, -1}}, {{1, 1}}, s, {}), "token id out of range");
  ScoreOptions o;
  o.top_n = 65;
  CHECK_THROWS(b->score({{1}}, {{1}}, s, o), "top_n");
  ModelBackend f16("synthetic:tiny:f16:seed=3", true);
  GenerationState s16 = f16.create_state(1);
  o = {};
  o.int8_head = true;
  CHECK_THROWS(f16.score({{1}}, {{1}}, s16, o), "int8 head");
  host_test::ScriptedBackend scripted(host_test::ScriptedBackend::script_for({1}, 8), "scripted");
  GenerationState none = scripted.create_state(1);
  CHECK_THROWS(scripted.score({{1}}, {{1}}, none, {}), "does not score");
}

// Texts of different lengths in one call: each gets what it gets alone (a text's chunks are the same, its neighbours change the shapes of
// the launches), over several chunks and with rows that drop out.
HOST_TEST(engine_scores_texts_of_any_lengths) {
  auto tok = std::make_shared<TrieTokenizer>();
  CHECK_EQ(tok->load(host_test::vocab_path()), 0);
  InferenceEngine engine(tiny(), tok, "tiny", 16);
  const std::string base = "The quick brown fox jumps over the lazy dog and runs on. ";
  const std::vector<std::string> texts = {base, "a", base + base + base, base.substr(0, 20)};
  ScoreOptions o;
  o.top_n = 1;
  const auto all = engine.score(texts, o);
  CHECK_EQ(all.size(), texts.size());
  for (std::size_t i = 0; i < texts.size(); ++i) {
    const auto one = engine.score({texts[i]}, o);
    CHECK(one[0].tokens == all[i].tokens);
    CHECK_EQ(int(all[i].tokens.size()), engine.count_tokens(texts[i]));
    CHECK_EQ(all[i].at.rows, int(all[i].tokens.size()));
    CHECK_EQ(all[i].at.logprob.size(), all[i].tokens.size());
    CHECK_EQ(all[i].at.entropy.size(), all[i].tokens.size());
    CHECK_EQ(all[i].at.top_ids.size(), all[i].tokens.size());
    CHECK_EQ(all[i].at.logprob[0], 0.0f);
    CHECK_EQ(all[i].at.top_ids[0], -1);
    double sum = 0;
    for (std::size_t t = 0; t < all[i].at.logprob.size(); ++t) {
      sum += all[i].at.logprob[t];
      CHECK_NEAR(all[i].at.logprob[t], one[0].at.logprob[t], 0.05);
      CHECK_NEAR(all[i].at.entropy[t], one[0].at.entropy[t], 0.05);
    }
    CHECK_NEAR(all[i].total(), sum, 1e-9);
  }
  CHECK(engine.score({}, o).empty());
  CHECK_THROWS(engine.score({""}, o), "prompt is empty");
  o.top_n = -1;
  CHECK_THROWS(engine.score({base}, o), "top_n");
  o.top_n = 65;
  CHECK_THROWS(engine.score({base}, o), "top_n");
}

int main(int argc, char** argv) { return host_test::run_all(argc, argv, true); }
