// Threads of one process that make decode graphs, copy, allocate and wait for the device at the same time.
#include <atomic>
#include <cmath>
#include <thread>

#include "rwkv_inference_engine.hpp"
#include "test_common.hpp"

using namespace rwkv7_server;

namespace {

constexpr int kVocab = 2048;

std::shared_ptr<ModelBackend> tiny() {
  static auto b = std::make_shared<ModelBackend>("synthetic:tiny:w8:seed=3", true);
  return b;
}

std::shared_ptr<TrieTokenizer> tokenizer() {
  static std::shared_ptr<TrieTokenizer> tok = [] {
    auto t = std::make_shared<TrieTokenizer>();
    if (t->load(host_test::vocab_path()) != kTokenizerSuccess) throw std::runtime_error("vocab load failed");
    return t;
  }();
  return tok;
}

// the logits of a few steps at several widths: states, logits and so decode graphs of their own
std::vector<float> widths(int first) {
  std::vector<float> out;
  for (int width = first; width < first + 6; ++width) {
    GenerationState s = tiny()->create_state(width);
    DeviceLogits logits;
    for (int step = 0; step < 3; ++step) {
      std::vector<int64_t> feed;
      for (int i = 0; i < width; ++i) feed.push_back((17 * i + 5 * step + first) % kVocab);
      tiny()->forward_decode(feed, s, logits);
    }
    const auto z = host_test::to_host<float>(logits.values);
    out.insert(out.end(), z.begin(), z.begin() + std::ptrdiff_t(width) * kVocab);
  }
  return out;
}

}  // namespace

// One thread makes decode graphs; others allocate, copy, clear and wait for the device
HOST_TEST(decode_graphs_beside_calls_of_other_threads) {
  const std::vector<float> want = widths(1);
  std::atomic<bool> done{false};
  std::vector<std::string> errors(3);
  std::vector<std::thread> threads;
  std::atomic<int> rounds{0};
  for (int i = 0; i < 2; ++i)
    threads.emplace_back([&, i] {
      try {
        std::vector<float> host(3000, float(i));
        while (!done) {
          GenerationState s = tiny()->create_state(2 + i);
          rwkv7_fast_v4::DeviceBuffer<float> b;
          host_test::to_device(host, b);
          if (host_test::to_host<float>(b)[2999] != float(i)) throw std::runtime_error("a copy came back changed");
          rwkv7_fast_v4::check_hip(rwkv_hip_device_sync(), "sync");
          tiny()->query_prefill_capacity(128);
          ++rounds;
        }
      } catch (const std::exception& e) {
        errors[i] = e.what();
      }
    });
  threads.emplace_back([&] {
    try {
      for (int k = 0; k < 12; ++k)
        if (widths(1) != want) throw std::runtime_error("other logits than alone");
    } catch (const std::exception& e) {
      errors[2] = e.what();
    }
    done = true;
  });
  for (auto& t : threads) t.join();
  for (const auto& e : errors)
    if (!e.empty()) FAIL_HERE(e);
  CHECK(rounds > 0);
}

HOST_TEST(decode_graphs_of_several_threads) {
  constexpr int kThreads = 3;
  std::vector<float> want[kThreads];
  for (int i = 0; i < kThreads; ++i) want[i] = widths(1 + 3 * i);
  std::vector<std::string> errors(kThreads);
  std::vector<std::thread> threads;
  for (int i = 0; i < kThreads; ++i)
    threads.emplace_back([&, i] {
      try {
        for (int k = 0; k < 6; ++k)
          if (widths(1 + 3 * i) != want[i]) throw std::runtime_error("other logits than alone");
      } catch (const std::exception& e) {
        errors[i] = e.what();
      }
    });
  for (auto& t : threads) t.join();
  for (const auto& e : errors)
    if (!e.empty()) FAIL_HERE(e);
}

HOST_TEST(branches_of_several_threads_at_once) {
  InferenceEngine engine(tiny(), tokenizer(), "tiny");
  constexpr int kThreads = 4;
  InferenceEngine::BranchOptions o[kThreads];
  std::vector<InferenceEngine::Branch> want[kThreads], got[kThreads][3];
  for (int i = 0; i < kThreads; ++i) {
    o[i].max_tokens = 12;
    o[i].seed = 20 + i;
    o[i].stop_tokens.clear();
    for (int t = 0; t < kVocab; t += 11) o[i].stop_tokens.push_back(t);
    o[i].draw.top_p = i % 2 ? 0.95 : 1.0;
    if (i > 1) o[i].draw.alpha_presence = 0.5;
    want[i] = engine.branch_generate("User: hi", 3 + 2 * i, o[i]);
  }
  std::vector<std::string> errors(kThreads);
  std::vector<std::thread> threads;
  for (int i = 0; i < kThreads; ++i)
    threads.emplace_back([&, i] {
      try {
        for (auto& g : got[i]) g = engine.branch_generate("User: hi", 3 + 2 * i, o[i]);
      } catch (const std::exception& e) {
        errors[i] = e.what();
      }
    });
  for (auto& t : threads) t.join();
  for (int i = 0; i < kThreads; ++i) {
    if (!errors[i].empty()) FAIL_HERE(errors[i]);
    for (const auto& g : got[i])
      for (size_t k = 0; k < want[i].size(); ++k) CHECK(g[k].tokens == want[i][k].tokens && g[k].logprobs == want[i][k].logprobs);
  }
}

int main(int argc, char** argv) { return host_test::run_all(argc, argv, true); }
