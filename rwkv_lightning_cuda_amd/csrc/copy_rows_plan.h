// In which order the rows of a call of copy_rows move: arithmetic on the row numbers alone, without a device.
#pragma once

#include <algorithm>
#include <cstdint>
#include <vector>

namespace rwkv {

constexpr int kMaxRowMoves = 512;  // of a call
constexpr int kMaxCopyRows = 65534;
constexpr int kMoveBatch = 8;      // moves whose loads are all made before the first of their stores
// A cycle that does not end in the batch it begins in takes a place more, and no two of them begin in one batch.
constexpr int kMaxOrdered = kMaxRowMoves * kMoveBatch / (kMoveBatch - 1) + 1;
constexpr uint16_t kRowZero = 65535;  // as a source: zeros
constexpr uint16_t kRowKept = 65534;  // as a destination: the value stays with the thread; as a source: that value again

struct RowMove {
  uint16_t to, from;
};

// Moves by source, so that a source is read once for all of its destinations: first[g] .. first[g + 1] are those of one source.
inline void group_moves(std::vector<RowMove>& moves, std::vector<uint16_t>& first) {
  std::stable_sort(moves.begin(), moves.end(), [](const RowMove& a, const RowMove& b) { return a.from < b.from; });
  first.clear();
  for (size_t i = 0; i < moves.size(); ++i)
    if (i == 0 || moves[i].from != moves[i - 1].from) first.push_back(static_cast<uint16_t>(i));
  first.push_back(static_cast<uint16_t>(moves.size()));
}

// Whether a destination is the source of another move
inline bool moves_depend(const std::vector<RowMove>& moves, int rows) {
  std::vector<char> is_source(rows, 0);
  for (const RowMove& m : moves)
    if (m.from != kRowZero) is_source[m.from] = 1;
  for (const RowMove& m : moves)
    if (is_source[m.to]) return true;
  return false;
}

// Moves inside one set of rows, every source as it is before the first of them, for a thread that makes them batch by batch: a row is
// overwritten in no earlier batch than the last that reads it.  Rows that nobody waits for go first; what is left are cycles: one that
// fits what is left of a batch is made as it is, another begins with one of its rows in the thread's keeping.
inline std::vector<RowMove> order_moves(const std::vector<RowMove>& moves, int rows) {
  std::vector<int> source_of(rows, -1), readers(rows, 0);
  for (const RowMove& m : moves) {
    source_of[m.to] = m.from;
    if (m.from != kRowZero) ++readers[m.from];
  }
  std::vector<RowMove> out;
  std::vector<int> ready;
  for (const RowMove& m : moves)
    if (readers[m.to] == 0) ready.push_back(m.to);
  for (size_t i = 0; i < ready.size(); ++i) {
    const int to = ready[i], from = source_of[to];
    out.push_back({static_cast<uint16_t>(to), static_cast<uint16_t>(from)});
    source_of[to] = -1;
    if (from != kRowZero && --readers[from] == 0 && source_of[from] >= 0) ready.push_back(from);
  }
  std::vector<uint16_t> cycle;
  for (const RowMove& m : moves) {
    if (source_of[m.to] < 0) continue;
    cycle.clear();
    for (int row = m.to; source_of[row] >= 0;) {
      const int from = source_of[row];
      cycle.push_back(static_cast<uint16_t>(row));
      source_of[row] = -1;
      row = from;
    }
    const size_t n = cycle.size();
    if (out.size() % kMoveBatch + n <= static_cast<size_t>(kMoveBatch)) {
      for (size_t i = 0; i < n; ++i) out.push_back({cycle[i], cycle[(i + 1) % n]});
    } else {
      out.push_back({kRowKept, cycle[0]});
      for (size_t i = 0; i + 1 < n; ++i) out.push_back({cycle[i], cycle[i + 1]});
      out.push_back({cycle[n - 1], kRowKept});
    }
  }
  return out;
}

}  // namespace rwkv
