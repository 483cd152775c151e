// How InferenceEngine::score splits its texts into calls of a backend: which tokens and targets arrive, how large the calls are and that
// every row comes back to its text.  No GPU: the backend here answers with numbers made of its state's lane, the token and the target.
#include <algorithm>

#include "rwkv_inference_engine.hpp"
#include "test_common.hpp"

using namespace rwkv7_server;

namespace {

// A lane's state is the number of tokens that it has seen; the log probability of a position is made of that, the token and the target.
class CountingBackend final : public IModelBackend {
 public:
  using Batch = std::vector<std::vector<int64_t>>;
  GenerationState create_state(int batch_size) const override {
    GenerationState s;
    s.batch_size = batch_size;
    seen.assign(batch_size, 0);
    most_texts = std::max(most_texts, batch_size);
    return s;
  }
  void copy_state_slice(const GenerationState& src, int so, GenerationState& dst, int dof, int count) const override {
    if (so != 0 || dof != 0 || count != dst.batch_size || count > src.batch_size) throw std::runtime_error("bad state slice");
    seen.assign(old.begin(), old.begin() + count);
  }
  TokenLogprobs score(const Batch& tokens, const Batch& targets, GenerationState& state, const ScoreOptions& o) const override {
    if (state.batch_size != int(tokens.size()) || targets.size() != tokens.size()) throw std::runtime_error("batch size");
    const int T = int(tokens[0].size());
    most_positions = std::max(most_positions, T * int(tokens.size()));
    longest = std::max(longest, T);
    TokenLogprobs out;
    out.rows = T * int(tokens.size());
    out.top_n = o.top_n;
    for (std::size_t b = 0; b < tokens.size(); ++b) {
      if (int(tokens[b].size()) != T || int(targets[b].size()) != T) throw std::runtime_error("not rectangular");
      for (int t = 0; t < T; ++t) {
        const float v = value(seen[b] + t, tokens[b][t], targets[b][t]);
        out.logprob.push_back(v);
        out.entropy.push_back(-v);
        for (int k = 0; k < o.top_n; ++k) {
          out.top_ids.push_back(int(targets[b][t]) + k);
          out.top_logprobs.push_back(v - float(k));
        }
      }
      seen[b] += T;
    }
    old = seen;
    return out;
  }
  static float value(int place, int64_t token, int64_t target) { return -float(place) - 0.25f * float(token % 61) - 16.0f * float(target % 13); }
  void forward_prefill(const Batch&, GenerationState&, DeviceLogits&) const override { throw std::runtime_error("not asked for"); }
  void forward_decode(const std::vector<int64_t>&, GenerationState&, DeviceLogits&) const override { throw std::runtime_error("not asked for"); }
  void copy_logits_slice(const DeviceLogits&, int, DeviceLogits&, int, int) const override { throw std::runtime_error("not asked for"); }
  PrefillCapacity query_prefill_capacity(int) const override { return {}; }
  int vocab_size() const override { return 65536; }
  const std::string& model_path() const override { return name_; }
  const std::string& model_name() const override { return name_; }

  mutable std::vector<int> seen, old;
  mutable int most_positions = 0, most_texts = 0, longest = 0;

 private:
  std::string name_ = "counting";
};

void check(const std::vector<std::string>& texts, int chunk, int top_n, CountingBackend* counts = nullptr) {
  auto tok = std::make_shared<TrieTokenizer>();
  CHECK_EQ(tok->load(host_test::vocab_path()), 0);
  auto backend = std::make_shared<CountingBackend>();
  InferenceEngine engine(backend, tok, "counting", chunk);
  ScoreOptions o;
  o.top_n = top_n;
  const auto scores = engine.score(texts, o);
  CHECK_EQ(scores.size(), texts.size());
  for (std::size_t i = 0; i < texts.size(); ++i) {
    const std::vector<int> ids = tok->encode(texts[i]);
    const TokenLogprobs& at = scores[i].at;
    CHECK_EQ(scores[i].tokens.size(), ids.size());
    CHECK_EQ(std::size_t(at.rows), ids.size());
    CHECK_EQ(at.logprob.size(), ids.size());
    CHECK_EQ(at.entropy.size(), ids.size());
    CHECK_EQ(at.top_ids.size(), ids.size() * top_n);
    CHECK_EQ(at.top_logprobs.size(), ids.size() * top_n);
    for (std::size_t t = 1; t < ids.size(); ++t) {
      const float want = CountingBackend::value(int(t) - 1, ids[t - 1], ids[t]);
      CHECK_EQ(scores[i].tokens[t], int64_t(ids[t]));
      CHECK_EQ(at.logprob[t], want);
      CHECK_EQ(at.entropy[t], -want);
      for (int k = 0; k < top_n; ++k) {
        CHECK_EQ(at.top_ids[t * top_n + k], ids[t] + k);
        CHECK_EQ(at.top_logprobs[t * top_n + k], want - float(k));
      }
    }
  }
  CHECK(backend->longest <= chunk);
  if (counts) *counts = *backend;
}

std::string text(int words) {
  const char* const some[] = {"quick ", "brown ", "fox ", "jumps ", "over ", "lazy ", "dog ", "1 ", "Z", "\n"};
  std::string s = "a";
  for (int i = 0; i < words; ++i) s += some[(i * 7 + words) % 10];
  return s;
}

}  // namespace

HOST_TEST(every_row_comes_back_to_its_text) {
  for (const int chunk : {1, 3, 16, 128})
    for (const int top_n : {0, 2}) check({text(5), "a", text(40), text(0), text(41), text(5), text(17)}, chunk, top_n);
}

HOST_TEST(texts_without_a_token_to_score) { check({"a", "b", "a"}, 16, 1); }

// However many texts there are, a call's positions and the states stay within bounds.
HOST_TEST(many_texts_go_in_groups) {
  std::vector<std::string> texts;
  for (int i = 0; i < 700; ++i) texts.push_back(text(i * 13 % 90));
  for (int i = 0; i < 600; ++i) texts.push_back(text(1));
  CountingBackend counts;
  check(texts, 128, 1, &counts);
  CHECK(counts.most_positions <= 8192);
  CHECK(counts.most_texts <= 256);
  check({text(900), text(1)}, 512, 0, &counts);
  CHECK(counts.longest > 128);
}

// A chunk that is longer than a whole call's positions goes one text at a time.
HOST_TEST(a_long_chunk_takes_one_text) {
  CountingBackend counts;
  check({text(9000), text(8900)}, 20000, 0, &counts);
  CHECK_EQ(counts.most_texts, 1);
}

int main(int argc, char** argv) { return host_test::run_all(argc, argv, false); }
