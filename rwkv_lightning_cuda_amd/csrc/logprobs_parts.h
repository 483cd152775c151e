// How a call of token_logprobs shares its rows out among blocks, and the workspace that takes: arithmetic on the sizes and the count of
// CUs alone, without a device.
#pragma once

#include <algorithm>
#include <cstddef>

#include "../../include/rwkv_hip.h"

namespace rwkv {

constexpr int kLogprobThreads = 256;  // of a block
constexpr int kMaxParts = 256;        // of a row

// Parts of a row: as many as bring the call to four blocks of 256 threads for every CU, each at least one batch long, and none where that
// is fewer than three (us with the join, fp32, 65536 entries: 64 rows in 16 parts 12.6, in 4 18.3; 200 rows in 5 20.8, whole 24.9; 400
// rows in 2 29.3, whole 27.9; 77 fp16 rows of 50277 in 7 12.3, in 13 13.6).
inline int logprob_parts(int rows, int V, int io, int cus) {
  const int batch = kLogprobThreads * (io == RWKV_IO_F16 ? 32 : 16);
  const int parts = std::min({4 * cus / rows, (V - 1) / batch + 1, kMaxParts});
  return parts < 3 ? 1 : parts;
}

// Candidates that a part hands on as they are, without sorting out its first top_n
constexpr int part_keys(int top_n) { return top_n > 0 ? 2 * top_n + 8 : 0; }

struct PartBytes {  // of the workspace, in this order
  size_t sums, ahead, token_logit, keys;
  size_t all() const { return sums + ahead + token_logit + keys; }
};
inline PartBytes part_bytes(int rows, int parts, int top_n) {
  const auto align = [](size_t n) { return (n + 15) / 16 * 16; };
  const size_t all = static_cast<size_t>(rows) * parts;
  return {all * 16, align(all * 4), align(static_cast<size_t>(rows) * 4), all * part_keys(top_n) * 8};
}

// of a call of `rows` rows (fp16 rows go in no more parts than fp32 ones)
inline size_t logprob_bytes(int rows, int V, int top_n, int cus) {
  const int parts = logprob_parts(rows, V, RWKV_IO_F32, cus);
  return parts == 1 ? 0 : part_bytes(rows, parts, top_n).all();
}

// of every call of up to `rows` rows: fewer of them may go in more parts
inline size_t most_logprob_bytes(int rows, int V, int top_n, int cus) {
  size_t most = 0;
  for (int r = std::min(rows, 4 * cus / 3); r > 0; --r) most = std::max(most, logprob_bytes(r, V, top_n, cus));  // (more rows: one part each)
  return most;
}

}  // namespace rwkv
