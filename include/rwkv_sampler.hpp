// Sampler host API, signature-compatible with the reference's include/rwkv_sampler.hpp.
#pragma once

#include <cstdint>
#include <vector>

#include "rwkv_server_backend.hpp"

namespace rwkv7_server {

struct SamplerPenaltyState {
  int batch_size = 0;
  int vocab_size = 0;
  rwkv7_fast_v4::DeviceBuffer<float> penalties;
  rwkv7_fast_v4::DeviceBuffer<float> probs;
  rwkv7_fast_v4::DeviceBuffer<int> outputs;
  rwkv7_fast_v4::DeviceBuffer<std::uint8_t> rand_states;  // unused: the generator is counter-based
  std::uint64_t seed = 0;   // Philox key
  std::uint64_t step = 0;   // Philox counter, advanced by every sampling call
};

// seed == 0 draws a seed from std::random_device and the clock as the reference does
// (src/rwkv_sampler.cpp:14-19); any other value makes the token stream reproducible.
SamplerPenaltyState make_sampler_penalties(int vocab_size, int batch_size = 1, std::uint64_t seed = 0);

// Streams: the sampling kernels run on the device's NULL stream and the token ids come back with a blocking copy,
// so the call returns with the ids on the host.  ModelBackend's forward calls run on per-session non-blocking
// streams and return only after their stream has drained, so logits handed from a forward call to the sampler on the
// same thread are complete, and the NULL stream never waits for another thread's forward.  Sampling calls of several
// threads queue behind one another on the NULL stream (each works on its own SamplerPenaltyState, so the results do
// not depend on the order); logits written by work still in flight on a stream of the caller's own must be
// synchronised by the caller first.
int sample_repetition_temperature_topk_topp(const DeviceLogits& logits, SamplerPenaltyState& penalties,
                                            const GenerateOptions& options);

std::vector<int> sample_batch_repetition_temperature_topk_topp(const DeviceLogits& logits,
                                                               SamplerPenaltyState& penalties,
                                                               const GenerateOptions& options);

// Log probability, entropy and rank of tokens[row] (-1: none) under each row of logits, with the top_n (0 .. 64) most probable entries:
// what a server returns as `logprobs` beside a sampled token.  Of the logits as they are, before penalties and temperature.  Streams as
// above.  No counterpart in the reference.
TokenLogprobs token_logprobs(const DeviceLogits& logits, const std::vector<int>& tokens, int top_n = 0);

// ---- a token per row from given random numbers, under options of the row's own (no counterpart in the reference) ----

// Filters that are off: top_k 0, top_p 1, min_p 0; temperature 0 takes the largest logit.  The penalties are the sampler's.
struct DrawOptions {
  double temperature = 1.0;
  int top_k = 0;
  double top_p = 1.0;
  double min_p = 0.0;  // entries less than this share as probable as the most probable one are not drawn
  double alpha_presence = 0.0;
  double alpha_frequency = 0.0;
  double alpha_decay = 1.0;
};

struct DrawState {
  int batch_size = 0;
  int vocab_size = 0;
  rwkv7_fast_v4::DeviceBuffer<float> penalties;  // [batch_size,vocab_size], empty without penalties
  rwkv7_fast_v4::DeviceBuffer<float> rows;       // options, numbers and answers of a call, 32 bits each
  rwkv7_fast_v4::DeviceBuffer<std::uint8_t> workspace;
  std::vector<float> host;
};

struct DrawnTokens {
  std::vector<int> tokens;      // -1: the row has no distribution (nothing but -infinity, a NaN)
  std::vector<float> logprobs;  // among the entries that the filters keep, at the row's temperature
};

DrawState make_draw_state(int vocab_size, int batch_size, bool with_penalties = true);

// Row i draws from logits row source[i] (empty: its own) with options[i] and uniform[i] in 0 .. 1; the penalties, if `state` has any, are
// brought up to date.  A row's token depends on nothing else.  Streams as for the sampler above.
DrawnTokens draw_tokens(const DeviceLogits& logits, const std::vector<DrawOptions>& options, const std::vector<float>& uniform, DrawState& state,
                        const std::vector<int>& source = {});

// The penalties of row rows[i] move to row to[i] (-1: none yet); as a sequence's state does with IModelBackend::copy_state_rows.  A row may be a
// destination once; up to 65534 rows, and 512 moves inside a state.  What is refused moves nothing.
void copy_draw_rows(const DrawState& src, const std::vector<int>& rows, DrawState& dst, const std::vector<int>& to);

// A uniform number in [0, 1) that depends on the three arguments alone, 24 bits of it: the number that step `step` of sequence `sequence`
// draws with, whatever else is in its batch.
float uniform_of(std::uint64_t seed, std::uint64_t sequence, std::uint64_t step);

}  // namespace rwkv7_server
