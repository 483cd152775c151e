// Sampler host wrapper (reference: src/rwkv_sampler.cpp:22-121): same argument checks and messages;
// the kernel launch goes through rwkv_hip_sample and the token ids come back with one blocking copy.
#include "rwkv_sampler.hpp"

#include <algorithm>
#include <chrono>
#include <cstring>
#include <random>
#include <stdexcept>

namespace rwkv7_server {
namespace {

std::uint64_t fresh_seed() {
  std::random_device rd;
  const auto now = static_cast<std::uint64_t>(std::chrono::high_resolution_clock::now().time_since_epoch().count());
  std::uint64_t s = (static_cast<std::uint64_t>(rd()) << 32) ^ static_cast<std::uint64_t>(rd()) ^ now;
  return s ? s : 1;
}

}  // namespace

SamplerPenaltyState make_sampler_penalties(int vocab_size, int batch_size, std::uint64_t seed) {
  if (vocab_size <= 0) throw std::runtime_error("invalid sampler vocab size");
  if (batch_size <= 0) throw std::runtime_error("invalid sampler batch size");
  SamplerPenaltyState state;
  state.batch_size = batch_size;
  state.vocab_size = vocab_size;
  const std::size_t n = static_cast<std::size_t>(batch_size) * vocab_size;
  state.penalties.resize(n, "alloc sampler penalties");
  state.probs.resize(n, "alloc sampler probs");
  state.outputs.resize(batch_size, "alloc sampler outputs");
  state.penalties.zero("zero sampler penalties");
  state.seed = seed ? seed : fresh_seed();
  state.step = 0;
  return state;
}

std::vector<int> sample_batch_repetition_temperature_topk_topp(const DeviceLogits& logits,
                                                               SamplerPenaltyState& penalties,
                                                               const GenerateOptions& options) {
  if (logits.rows <= 0) throw std::runtime_error("sampler expects at least one logits row");
  if (logits.vocab_size <= 0 || logits.values.p == nullptr) throw std::runtime_error("empty device logits");
  if (penalties.vocab_size != logits.vocab_size)
    throw std::runtime_error("sampler logits size does not match sampler state");
  if (penalties.batch_size != logits.rows)
    throw std::runtime_error("sampler batch size does not match logits rows");

  const bool use_penalty = options.alpha_presence != 0.0 || options.alpha_frequency != 0.0;
  const int rc = rwkv_hip_sample(nullptr, logits.rows, logits.vocab_size, logits.values.p,
                                 use_penalty ? penalties.penalties.p : nullptr, penalties.probs.p, penalties.outputs.p,
                                 options.alpha_presence, options.alpha_frequency, options.alpha_decay,
                                 options.temperature, options.top_k, options.top_p, penalties.seed, penalties.step++);
  if (rc != RWKV_OK) throw std::invalid_argument(rwkv_hip_last_error());
  std::vector<int> tokens(static_cast<std::size_t>(logits.rows));
  rwkv7_fast_v4::check_hip(rwkv_hip_memcpy_d2h(tokens.data(), penalties.outputs.p, tokens.size() * sizeof(int)),
                           "copy sampled tokens to host");
  return tokens;
}

int sample_repetition_temperature_topk_topp(const DeviceLogits& logits, SamplerPenaltyState& penalties,
                                            const GenerateOptions& options) {
  if (logits.rows != 1) throw std::runtime_error("sampler currently expects a single logits row");
  return sample_batch_repetition_temperature_topk_topp(logits, penalties, options).front();
}

TokenLogprobs token_logprobs(const DeviceLogits& logits, const std::vector<int>& tokens, int top_n) {
  using rwkv7_fast_v4::DeviceBuffer;
  using rwkv7_fast_v4::check_hip;
  if (logits.rows <= 0) throw std::runtime_error("token_logprobs expects at least one logits row");
  if (logits.vocab_size <= 0 || logits.values.p == nullptr) throw std::runtime_error("empty device logits");
  if (static_cast<int>(tokens.size()) != logits.rows) throw std::runtime_error("token_logprobs expects a token per logits row");
  for (const int t : tokens)
    if (t < -1 || t >= logits.vocab_size) throw std::runtime_error("token id out of range");
  std::size_t need = 0;
  if (rwkv_hip_token_logprobs_workspace(logits.rows, logits.vocab_size, top_n, &need) != RWKV_OK) throw std::invalid_argument(rwkv_hip_last_error());
  const std::size_t rows = tokens.size(), top = rows * top_n;
  // one buffer of 32-bit values: tokens, log probabilities, entropies, ranks, the alternatives' log probabilities and ids
  DeviceBuffer<float> dev;
  DeviceBuffer<std::uint8_t> workspace;
  dev.resize_recycled(4 * rows + 2 * top, "alloc log probabilities");
  if (need) workspace.resize_recycled(need, "alloc log probability workspace");
  check_hip(rwkv_hip_memcpy_h2d(dev.p, tokens.data(), rows * sizeof(int)), "copy tokens");
  const int rc = rwkv_hip_token_logprobs(nullptr, logits.rows, logits.vocab_size, RWKV_IO_F32, logits.values.p, logits.vocab_size, dev.p, top_n,
                                         dev.p + rows, dev.p + 2 * rows, dev.p + 3 * rows, top ? dev.p + 4 * rows + top : nullptr,
                                         top ? dev.p + 4 * rows : nullptr, workspace.p, need);
  if (rc != RWKV_OK) throw std::invalid_argument(rwkv_hip_last_error());
  TokenLogprobs out;
  out.rows = logits.rows;
  out.top_n = top_n;
  out.logprob.resize(rows);
  out.entropy.resize(rows);
  out.rank.resize(rows);
  out.top_logprobs.resize(top);
  out.top_ids.resize(top);
  check_hip(rwkv_hip_memcpy_d2h(out.logprob.data(), dev.p + rows, rows * sizeof(float)), "copy log probabilities");
  check_hip(rwkv_hip_memcpy_d2h(out.entropy.data(), dev.p + 2 * rows, rows * sizeof(float)), "copy entropies");
  check_hip(rwkv_hip_memcpy_d2h(out.rank.data(), dev.p + 3 * rows, rows * sizeof(int)), "copy ranks");
  if (top) {
    check_hip(rwkv_hip_memcpy_d2h(out.top_logprobs.data(), dev.p + 4 * rows, top * sizeof(float)), "copy alternatives");
    check_hip(rwkv_hip_memcpy_d2h(out.top_ids.data(), dev.p + 4 * rows + top, top * sizeof(int)), "copy alternatives");
  }
  return out;
}

DrawState make_draw_state(int vocab_size, int batch_size, bool with_penalties) {
  if (vocab_size <= 0) throw std::runtime_error("invalid sampler vocab size");
  if (batch_size <= 0) throw std::runtime_error("invalid sampler batch size");
  DrawState state;
  state.batch_size = batch_size;
  state.vocab_size = vocab_size;
  std::size_t need = 0;
  if (rwkv_hip_draw_tokens_workspace(batch_size, vocab_size, &need) != RWKV_OK) throw std::invalid_argument(rwkv_hip_last_error());
  if (with_penalties) {
    state.penalties.resize_recycled(static_cast<std::size_t>(batch_size) * vocab_size, "alloc draw penalties");
    state.penalties.zero("zero draw penalties");
  }
  state.rows.resize_recycled(11 * static_cast<std::size_t>(batch_size), "alloc draw rows");
  state.workspace.resize_recycled(need, "alloc draw workspace");
  return state;
}

DrawnTokens draw_tokens(const DeviceLogits& logits, const std::vector<DrawOptions>& options, const std::vector<float>& uniform, DrawState& state,
                        const std::vector<int>& source) {
  using rwkv7_fast_v4::check_hip;
  if (logits.rows <= 0) throw std::runtime_error("sampler expects at least one logits row");
  if (logits.vocab_size <= 0 || logits.values.p == nullptr) throw std::runtime_error("empty device logits");
  if (state.vocab_size != logits.vocab_size) throw std::runtime_error("sampler logits size does not match sampler state");
  const std::size_t rows = options.size();
  if (rows != static_cast<std::size_t>(state.batch_size)) throw std::runtime_error("sampler batch size does not match its options");
  if (uniform.size() != rows) throw std::runtime_error("a random number for every row");
  if (source.empty() ? static_cast<std::size_t>(logits.rows) != rows : source.size() != rows)
    throw std::runtime_error("sampler batch size does not match logits rows");
  for (const int s : source)
    if (s < 0 || s >= logits.rows) throw std::runtime_error("logits row out of range");
  for (std::size_t i = 0; i < rows; ++i) {
    if (!(options[i].temperature >= 0.0) || options[i].top_p != options[i].top_p || options[i].min_p != options[i].min_p)
      throw std::invalid_argument("sampler options are negative or not a number");
    if (!(uniform[i] >= 0.0f && uniform[i] <= 1.0f)) throw std::invalid_argument("random number outside 0 .. 1");
  }
  // nine tensors of `rows` values, then the two of the answer
  state.host.resize(9 * rows);
  float* at = state.host.data();
  for (std::size_t i = 0; i < rows; ++i) {
    const DrawOptions& o = options[i];
    const float values[9] = {static_cast<float>(o.temperature), 0.0f, static_cast<float>(o.top_p), static_cast<float>(o.min_p), uniform[i],
                             static_cast<float>(o.alpha_presence), static_cast<float>(o.alpha_frequency), static_cast<float>(o.alpha_decay), 0.0f};
    for (int k = 0; k < 9; ++k) at[k * rows + i] = values[k];
    std::memcpy(at + rows + i, &o.top_k, sizeof(int));
    if (!source.empty()) std::memcpy(at + 8 * rows + i, &source[i], sizeof(int));
  }
  check_hip(rwkv_hip_memcpy_h2d(state.rows.p, at, 9 * rows * sizeof(float)), "copy draw options");
  float* d = state.rows.p;
  const bool penalised = state.penalties.p != nullptr;
  const int rc = rwkv_hip_draw_tokens(nullptr, static_cast<int>(rows), logits.vocab_size, RWKV_IO_F32, logits.values.p, logits.vocab_size, logits.rows,
                                      source.empty() ? nullptr : d + 8 * rows, d, d + rows, d + 2 * rows, d + 3 * rows, d + 4 * rows,
                                      state.penalties.p, penalised ? d + 5 * rows : nullptr, penalised ? d + 6 * rows : nullptr,
                                      penalised ? d + 7 * rows : nullptr, state.penalties.p, d + 9 * rows, d + 10 * rows, state.workspace.p,
                                      state.workspace.n);
  if (rc != RWKV_OK) throw std::invalid_argument(rwkv_hip_last_error());
  std::vector<float> answer(2 * rows);
  check_hip(rwkv_hip_memcpy_d2h(answer.data(), d + 9 * rows, 2 * rows * sizeof(float)), "copy drawn tokens to host");
  DrawnTokens out;
  out.tokens.resize(rows);
  std::memcpy(out.tokens.data(), answer.data(), rows * sizeof(int));
  out.logprobs.assign(answer.begin() + rows, answer.end());
  return out;
}

void copy_draw_rows(const DrawState& src, const std::vector<int>& rows, DrawState& dst, const std::vector<int>& to) {
  using rwkv7_fast_v4::check_hip;
  if (src.vocab_size != dst.vocab_size || (src.penalties.p == nullptr) != (dst.penalties.p == nullptr))
    throw std::runtime_error("draw states do not match");
  if (rows.size() != to.size()) throw std::runtime_error("as many draw rows as places for them");
  if (&src == &dst && rows.size() > 512) throw std::runtime_error("more than 512 rows inside a draw state");
  if (std::max(src.batch_size, dst.batch_size) > 65534) throw std::runtime_error("more than 65534 rows of a draw state");
  std::vector<char> taken(dst.batch_size, 0);
  for (std::size_t i = 0; i < rows.size(); ++i) {  // (over all launches, ahead of the first)
    if (rows[i] < -1 || rows[i] >= src.batch_size || to[i] < 0 || to[i] >= dst.batch_size) throw std::runtime_error("draw row out of range");
    if (taken[to[i]]) throw std::runtime_error("two draw rows for one place");
    taken[to[i]] = 1;
  }
  if (src.penalties.p == nullptr) return;
  const std::int64_t planes = 1, bytes = src.vocab_size * static_cast<std::int64_t>(sizeof(float));
  void* to_tensor = dst.penalties.p;
  const void* from_tensor = src.penalties.p;
  for (std::size_t i = 0; i < rows.size(); i += 512) {
    const int n = static_cast<int>(std::min<std::size_t>(512, rows.size() - i));
    check_hip(rwkv_hip_copy_rows(nullptr, 1, &to_tensor, &from_tensor, &planes, &bytes, dst.batch_size, src.batch_size, n, to.data() + i, rows.data() + i),
              "copy draw rows");
  }
  check_hip(rwkv_hip_stream_sync(nullptr), "copy draw rows");
}

// The finaliser of SplitMix64 (Steele, Lea and Flood, 2014) over the three numbers, one after the other.
float uniform_of(std::uint64_t seed, std::uint64_t sequence, std::uint64_t step) {
  std::uint64_t x = seed;
  for (const std::uint64_t part : {sequence, step}) {
    x += 0x9E3779B97F4A7C15ull * (part + 1);
    x = (x ^ (x >> 30)) * 0xBF58476D1CE4E5B9ull;
    x = (x ^ (x >> 27)) * 0x94D049BB133111EBull;
    x ^= x >> 31;
  }
  return static_cast<float>(x >> 40) * (1.0f / 16777216.0f);
}

}  // namespace rwkv7_server
