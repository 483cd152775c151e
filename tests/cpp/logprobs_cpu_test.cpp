// The workspaces of the log probabilities for any count of CUs (a card may be partitioned).  No GPU.
#include "../../rwkv_lightning_cuda_amd/csrc/logprobs_parts.h"
#include "test_common.hpp"

using namespace rwkv;

namespace {
constexpr int kCus[] = {8, 32, 38, 64, 128, 191, 192, 256, 304};
constexpr int kVocabs[] = {1, 2048, 8193, 12288, 12289, 50277, 65536, 262144, 1048576};
}  // namespace

// What is made for blocks of up to so many rows holds every shorter block's parts too, of which a row may have more.
HOST_TEST(a_blocks_workspace_serves_every_shorter_block) {
  for (const int cus : kCus)
    for (const int V : kVocabs)
      for (const int top_n : {0, 1, 5, 64})
        for (const int block : {1, 2, 64, 255, 256, 300, 341, 342, 2048}) {
          const size_t have = most_logprob_bytes(block, V, top_n, cus);
          for (int rows = 1; rows <= block; ++rows)
            if (logprob_bytes(rows, V, top_n, cus) > have) FAIL_HERE(cus << " CUs, V " << V << ", top_n " << top_n << ": " << rows << " rows of " << block);
        }
}

HOST_TEST(fp16_rows_need_no_more) {
  for (const int cus : kCus)
    for (const int V : kVocabs)
      for (int rows = 1; rows <= 600; ++rows) CHECK(logprob_parts(rows, V, RWKV_IO_F16, cus) <= logprob_parts(rows, V, RWKV_IO_F32, cus));
}

// A block per CU and more of them where there are few rows; never more than a row can have, never few that do not pay for the join.
HOST_TEST(parts_of_a_row) {
  for (const int cus : kCus)
    for (const int V : kVocabs)
      for (int rows = 1; rows <= 2048; ++rows) {
        const int parts = logprob_parts(rows, V, RWKV_IO_F32, cus);
        CHECK(parts == 1 || (parts >= 3 && parts <= kMaxParts && parts * rows <= 4 * cus && (parts - 1) * 4096 < V));
      }
  CHECK_EQ(logprob_parts(1, 65536, RWKV_IO_F32, 256), 16);
  CHECK_EQ(logprob_parts(44, 65536, RWKV_IO_F32, 32), 1);
  CHECK_EQ(logprob_parts(1, 1, RWKV_IO_F32, 256), 1);
}

int main(int argc, char** argv) { return host_test::run_all(argc, argv, false); }
