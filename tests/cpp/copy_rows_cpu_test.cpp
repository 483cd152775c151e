// The order in which copy_rows makes moves inside one set of rows, checked by making them batch by batch on numbers.  No GPU.
#include "../../rwkv_lightning_cuda_amd/csrc/copy_rows_plan.h"

#include <numeric>
#include <random>

#include "test_common.hpp"

using namespace rwkv;

namespace {

// what a thread of the kernel does with its unit of every row
std::vector<int> run(const std::vector<RowMove>& order, std::vector<int> rows) {
  int kept = -77;
  for (size_t first = 0; first < order.size(); first += kMoveBatch) {
    const size_t end = std::min(first + kMoveBatch, order.size());
    std::vector<int> v;
    for (size_t i = first; i < end; ++i) v.push_back(order[i].from == kRowKept ? kept : order[i].from == kRowZero ? 0 : rows[order[i].from]);
    for (size_t i = first; i < end; ++i) {
      if (order[i].to == kRowKept) kept = v[i - first];
      else rows[order[i].to] = v[i - first];
    }
  }
  return rows;
}

void check(const std::vector<RowMove>& moves, int rows) {
  std::vector<int> before(rows);
  std::iota(before.begin(), before.end(), 1000);
  std::vector<int> want = before;
  for (const RowMove& m : moves) want[m.to] = m.from == kRowZero ? 0 : before[m.from];
  const std::vector<RowMove> order = order_moves(moves, rows);
  CHECK(order.size() <= static_cast<size_t>(kMaxOrdered));
  CHECK(run(order, before) == want);
}

RowMove move(int to, int from) { return {static_cast<uint16_t>(to), static_cast<uint16_t>(from)}; }

}  // namespace

HOST_TEST(chains_and_cycles_of_every_length) {
  for (int n = 2; n <= 40; ++n)
    for (int lead = 0; lead < 9; ++lead) {
      std::vector<RowMove> cycle, chain;
      for (int i = 0; i < lead; ++i) cycle.push_back(move(100 + 2 * i, 101 + 2 * i));  // (where in a batch the cycle begins)
      for (int i = 0; i < n; ++i) cycle.push_back(move(i, (i + 1) % n));
      check(cycle, 200);
      for (int i = 0; i < n; ++i) chain.push_back(move(i, i + 1));
      check(chain, 200);
      for (int i = 0; i < n; ++i) chain[i] = move(n - i, n - i - 1);
      check(chain, 200);
    }
}

HOST_TEST(any_moves_keep_what_the_rows_held) {
  std::mt19937 g(7);
  for (int trial = 0; trial < 4000; ++trial) {
    const int rows = 2 + g() % (trial % 50 == 0 ? 512 : 40);
    std::vector<int> to(rows), from(rows);
    std::iota(to.begin(), to.end(), 0);
    std::shuffle(to.begin(), to.end(), g);
    from = to;
    std::shuffle(from.begin(), from.end(), g);  // a permutation
    std::vector<RowMove> moves;
    const unsigned kind = g() % 3;
    for (int i = 0, n = 1 + g() % rows; i < n; ++i) {
      int source = kind == 0 ? from[i] : static_cast<int>(g() % rows);
      if (kind == 2 && g() % 4 == 0) source = kRowZero;
      if (source != to[i]) moves.push_back(move(to[i], source));
    }
    check(moves, rows);
  }
}

HOST_TEST(the_largest_call_fits_whatever_the_cycles) {
  std::mt19937 g(3);
  for (int longest = 2; longest <= 20; ++longest)
    for (int trial = 0; trial < 20; ++trial) {
      std::vector<RowMove> moves;
      int row = 0;
      while (row + 1 < kMaxRowMoves) {
        const int n = std::min<int>(2 + g() % (longest - 1), kMaxRowMoves - row);
        if (n < 2) break;
        for (int i = 0; i < n; ++i) moves.push_back(move(row + i, row + (i + 1) % n));
        row += n;
      }
      check(moves, kMaxRowMoves);
    }
}

HOST_TEST(groups_hold_every_move_once) {
  std::vector<RowMove> moves = {move(5, 1), move(2, 0), move(7, 1), move(1, kRowZero), move(3, 0), move(9, kRowZero)};
  std::vector<uint16_t> first;
  group_moves(moves, first);
  CHECK(first == (std::vector<uint16_t>{0, 2, 4, 6}));
  CHECK(moves[0].to == 2 && moves[1].to == 3 && moves[2].to == 5 && moves[3].to == 7 && moves[4].to == 1 && moves[5].to == 9);
  CHECK(moves_depend(moves, 10));
  CHECK(!moves_depend({move(3, 0), move(4, 0), move(5, kRowZero)}, 10));
}

int main(int argc, char** argv) { return host_test::run_all(argc, argv, false); }
