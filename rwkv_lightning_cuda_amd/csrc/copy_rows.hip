// Rows of several tensors copied, forked, exchanged and cleared in one launch: what the cache of generation states needs when sequences
// branch, end and make room.  The reference moves a state with a copy for every layer and tensor (copy_state_slice,
// src/rwkv7_fast_v4.cu:1421-1504) and has no fork.
//
// A tensor is [planes, rows, row_bytes]; the rows of a move are the same in every plane.  Bound by memory: every source row is read once
// for all of its destinations, every destination written once.
#include <new>

#include "copy_rows_plan.h"
#include "ops.h"

namespace rwkv {

namespace {

constexpr int kThreads = 256;
constexpr int kMaxTensors = 8;

struct RowTensor {
  const char* src;
  char* dst;
  int64_t src_plane, dst_plane;  // bytes between planes
  int64_t row_bytes;
  int first_block, blocks_per_plane;
  int unit;  // bytes of an access: 16, 4, 2 or 1
};

struct RowTensors {
  RowTensor of[kMaxTensors];
  int count;
};

struct GroupArgs {  // moves that do not depend on one another, by source
  RowTensors tensors;
  RowMove moves[kMaxRowMoves];
  uint16_t first[kMaxRowMoves + 1];
};

struct OrderArgs {
  RowTensors tensors;
  int n;
  RowMove moves[kMaxOrdered];
};

static_assert(sizeof(GroupArgs) <= 4096 && sizeof(OrderArgs) <= 4096, "kernel arguments");

// The tensor of a block, its plane and its first byte in a row
struct Place {
  RowTensor t;
  int64_t plane, byte;
};
__device__ __forceinline__ Place place_of_block(const RowTensors& all, int per_thread) {
  const int block = blockIdx.x;
  int i = 0;
  while (i + 1 < all.count && block >= all.of[i + 1].first_block) ++i;
  Place p;
  p.t = all.of[i];
  const int local = block - p.t.first_block;
  p.plane = local / p.t.blocks_per_plane;
  p.byte = static_cast<int64_t>(local % p.t.blocks_per_plane) * kThreads * per_thread * p.t.unit;
  return p;
}

template <typename U, bool NT>
__device__ __forceinline__ U load_unit(const char* p) {
  if constexpr (NT) return __builtin_nontemporal_load(reinterpret_cast<const U*>(p));
  else return *reinterpret_cast<const U*>(p);
}
template <typename U, bool NT>
__device__ __forceinline__ void store_unit(char* p, U v) {
  if constexpr (NT) __builtin_nontemporal_store(v, reinterpret_cast<U*>(p));
  else *reinterpret_cast<U*>(p) = v;
}

// A block takes kThreads * PER units of one source row and writes them to all destinations of that source: a row that forks is read once, and
// its copies leave from registers.  Bound by memory: 32 of 64 fp32 states of the 7.2B shape to a narrower batch (2.2 GB) 425 us, 5.2 TB/s, where
// a copy of 2 GiB with the same loads and stores reaches 5.9; one state of the 0.1B shape (2.4 MB) is a launch.
template <typename U, int PER, bool NT>
__device__ __forceinline__ void copy_group(const GroupArgs& a, const Place& p) {
  const int begin = a.first[blockIdx.y], end = a.first[blockIdx.y + 1];
  const int from = a.moves[begin].from;
  const int64_t at = p.byte + static_cast<int64_t>(threadIdx.x) * sizeof(U);
  const char* src = p.t.src + p.plane * p.t.src_plane + from * p.t.row_bytes;
  char* plane = p.t.dst + p.plane * p.t.dst_plane;
  U v[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int64_t byte = at + static_cast<int64_t>(i) * kThreads * sizeof(U);
    v[i] = U{};
    if (from != kRowZero && byte < p.t.row_bytes) v[i] = load_unit<U, NT>(src + byte);
  }
  for (int m = begin; m < end; ++m) {
    char* dst = plane + a.moves[m].to * p.t.row_bytes;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int64_t byte = at + static_cast<int64_t>(i) * kThreads * sizeof(U);
      if (byte < p.t.row_bytes) store_unit<U, NT>(dst + byte, v[i]);
    }
  }
}

template <int PER, bool NT>
__global__ __launch_bounds__(kThreads) void copy_rows_kernel(GroupArgs a) {
  const Place p = place_of_block(a.tensors, PER);
  switch (p.t.unit) {
    case 16: return copy_group<uint4_t, PER, NT>(a, p);
    case 4: return copy_group<uint32_t, PER, NT>(a, p);
    case 2: return copy_group<uint16_t, PER, NT>(a, p);
    default: return copy_group<uint8_t, PER, NT>(a, p);
  }
}

// Moves inside one set of rows that overwrite one another's sources.  A thread has one unit of every row to itself and makes the moves
// in order, kMoveBatch loads ahead of as many stores: no other thread reads or writes its bytes, so nothing has to wait.  48 fp32 states of the
// 7.2B shape in another order (3.1 GB) 659 us, 4.7 TB/s; nine neighbours a place on (0.61 GB) 111; 29 fp16 ones of the 1.5B shape (0.38 GB) 50.  Past
// the caches, as above: 641, 118 and 74.
template <typename U>
__device__ __forceinline__ void move_in_order(const OrderArgs& a, const Place& p) {
  const int64_t at = p.byte + static_cast<int64_t>(threadIdx.x) * sizeof(U);
  if (at >= p.t.row_bytes) return;
  char* rows = p.t.dst + p.plane * p.t.dst_plane + at;
  U kept = {};
  for (int first = 0; first < a.n; first += kMoveBatch) {
    U v[kMoveBatch];
#pragma unroll
    for (int i = 0; i < kMoveBatch; ++i) {
      v[i] = U{};
      if (first + i < a.n) {
        const RowMove m = a.moves[first + i];
        if (m.from == kRowKept) v[i] = kept;
        else if (m.from != kRowZero) v[i] = *reinterpret_cast<const U*>(rows + m.from * p.t.row_bytes);
      }
    }
#pragma unroll
    for (int i = 0; i < kMoveBatch; ++i) {
      if (first + i < a.n) {
        const RowMove m = a.moves[first + i];
        if (m.to == kRowKept) kept = v[i];
        else *reinterpret_cast<U*>(rows + m.to * p.t.row_bytes) = v[i];
      }
    }
  }
}

__global__ __launch_bounds__(kThreads) void move_rows_kernel(OrderArgs a) {
  const Place p = place_of_block(a.tensors, 1);
  switch (p.t.unit) {
    case 16: return move_in_order<uint4_t>(a, p);
    case 4: return move_in_order<uint32_t>(a, p);
    case 2: return move_in_order<uint16_t>(a, p);
    default: return move_in_order<uint8_t>(a, p);
  }
}

struct Range {
  uintptr_t begin, end;
  bool meets(const Range& o) const { return begin < o.end && o.begin < end; }
};

// Blocks of the tensors with so many units to a thread; 0 where they are too many for a launch
int64_t lay_out_blocks(RowTensors& t, const int64_t* planes, int per_thread) {
  int64_t blocks = 0;
  for (int i = 0; i < t.count; ++i) {
    const int64_t bytes = static_cast<int64_t>(kThreads) * per_thread * t.of[i].unit;
    const int64_t per_plane = (t.of[i].row_bytes + bytes - 1) / bytes;
    t.of[i].first_block = static_cast<int>(blocks);
    t.of[i].blocks_per_plane = static_cast<int>(std::min<int64_t>(per_plane, INT32_MAX));
    // (a launch has less than 2^32 threads)
    if (per_plane >= (int64_t{1} << 24) || planes[i] >= (int64_t{1} << 24)) return 0;
    blocks += per_plane * planes[i];
    if (blocks >= (int64_t{1} << 24)) return 0;
  }
  return blocks;
}

}  // namespace

int copy_rows_launch(hipStream_t st, int tensors, void* const* dst, const void* const* src, const int64_t* planes, const int64_t* row_bytes,
                     int dst_rows, int src_rows, int n, const int32_t* to, const int32_t* from) {
  RWKV_REQUIRE(tensors > 0 && tensors <= kMaxTensors, "copy_rows: 1 .. %d tensors, got %d", kMaxTensors, tensors);
  RWKV_REQUIRE(dst && src && planes && row_bytes, "copy_rows: NULL list of tensors");
  RWKV_REQUIRE(dst_rows > 0 && dst_rows <= kMaxCopyRows && src_rows > 0 && src_rows <= kMaxCopyRows, "copy_rows: 1 .. %d rows, got %d and %d",
               kMaxCopyRows, dst_rows, src_rows);
  RWKV_REQUIRE(n >= 0 && n <= kMaxRowMoves, "copy_rows: up to %d moves, got %d", kMaxRowMoves, n);
  RWKV_REQUIRE(n == 0 || (to && from), "copy_rows: NULL list of rows");

  std::vector<Range> written, read;
  int in_place = 0;
  RowTensors t = {};
  t.count = tensors;
  int64_t plane_bytes = 0;
  for (int i = 0; i < tensors; ++i) {
    RWKV_REQUIRE(dst[i] && src[i], "copy_rows: tensor %d is NULL", i);
    RWKV_REQUIRE(planes[i] > 0 && row_bytes[i] > 0, "copy_rows: tensor %d has %lld planes and rows of %lld bytes", i, static_cast<long long>(planes[i]),
                 static_cast<long long>(row_bytes[i]));
    const int64_t most = int64_t{1} << 46;
    RWKV_REQUIRE(row_bytes[i] <= most / kMaxCopyRows && planes[i] <= most / (row_bytes[i] * std::max(dst_rows, src_rows)),
                 "copy_rows: tensor %d is larger than any memory", i);
    const uintptr_t d = reinterpret_cast<uintptr_t>(dst[i]), s = reinterpret_cast<uintptr_t>(src[i]);
    written.push_back({d, d + static_cast<uintptr_t>(planes[i] * dst_rows * row_bytes[i])});
    read.push_back({s, s + static_cast<uintptr_t>(planes[i] * src_rows * row_bytes[i])});
    in_place += d == s;
    plane_bytes += planes[i] * row_bytes[i];
    const uintptr_t bits = d | s | static_cast<uintptr_t>(row_bytes[i]);
    t.of[i] = {static_cast<const char*>(src[i]), static_cast<char*>(dst[i]), src_rows * row_bytes[i], dst_rows * row_bytes[i], row_bytes[i], 0, 0,
               (bits & 15) == 0 ? 16 : (bits & 3) == 0 ? 4 : (bits & 1) == 0 ? 2 : 1};
  }
  RWKV_REQUIRE(in_place == 0 || in_place == tensors, "copy_rows: tensors that move in place beside tensors that do not");
  RWKV_REQUIRE(!in_place || dst_rows == src_rows, "copy_rows: in place, but %d and %d rows", dst_rows, src_rows);
  for (int i = 0; i < tensors; ++i)
    for (int j = 0; j < i; ++j) RWKV_REQUIRE(!written[i].meets(written[j]), "copy_rows: destinations %d and %d overlap", j, i);
  for (int i = 0; i < tensors; ++i)
    for (int j = 0; j < tensors; ++j)
      RWKV_REQUIRE((in_place && i == j) || !written[i].meets(read[j]), "copy_rows: destination %d overlaps source %d", i, j);

  std::vector<RowMove> moves;
  std::vector<char> taken(dst_rows, 0);
  for (int i = 0; i < n; ++i) {
    RWKV_REQUIRE(to[i] >= 0 && to[i] < dst_rows, "copy_rows: move %d goes to row %d of %d", i, to[i], dst_rows);
    RWKV_REQUIRE(from[i] >= -1 && from[i] < src_rows, "copy_rows: move %d comes from row %d of %d", i, from[i], src_rows);
    RWKV_REQUIRE(!taken[to[i]], "copy_rows: two moves go to row %d", to[i]);
    taken[to[i]] = 1;
    if (in_place && to[i] == from[i]) continue;
    moves.push_back({static_cast<uint16_t>(to[i]), from[i] < 0 ? kRowZero : static_cast<uint16_t>(from[i])});
  }
  if (moves.empty()) return RWKV_OK;

  if (in_place && moves_depend(moves, dst_rows)) {
    OrderArgs a;
    a.tensors = t;
    const int64_t blocks = lay_out_blocks(a.tensors, planes, 1);
    RWKV_REQUIRE(blocks > 0, "copy_rows: too large for one call");
    const std::vector<RowMove> order = order_moves(moves, dst_rows);
    RWKV_REQUIRE(order.size() <= static_cast<size_t>(kMaxOrdered), "copy_rows: %zu ordered moves", order.size());
    a.n = static_cast<int>(order.size());
    std::copy(order.begin(), order.end(), a.moves);
    hipLaunchKernelGGL(move_rows_kernel, dim3(static_cast<unsigned>(blocks)), dim3(kThreads), 0, st, a);
  } else {
    GroupArgs a;
    std::vector<uint16_t> first;
    group_moves(moves, first);
    std::copy(moves.begin(), moves.end(), a.moves);
    std::copy(first.begin(), first.end(), a.first);
    a.tensors = t;
    // us with 1 / 2 / 4 / 8 units a thread: a fp16 state of the 7.2B shape to fifteen rows 57 / 58 / 63 / 67, half of 64 fp32 ones to a
    // narrower batch 438 / 417 / 439 / 668.  Past the caches where more is moved than the last of them holds: nine of 48 such states to
    // other places and as many cleared (0.93 GB) 168 instead of 189; three states of the 1.5B shape to eleven (0.14 GB) 28 instead of 26.
    constexpr int kPer = 2;
    const int64_t blocks = lay_out_blocks(a.tensors, planes, kPer);
    RWKV_REQUIRE(blocks > 0, "copy_rows: too large for one call");
    const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>(first.size() - 1));
    const bool past = (moves.size() + first.size() - 1) * static_cast<double>(plane_bytes) >= 256.0 * (1 << 20);
    if (past) hipLaunchKernelGGL((copy_rows_kernel<kPer, true>), grid, dim3(kThreads), 0, st, a);
    else hipLaunchKernelGGL((copy_rows_kernel<kPer, false>), grid, dim3(kThreads), 0, st, a);
  }
  RWKV_LAUNCH_CHECK();
  return RWKV_OK;
}

}  // namespace rwkv

using namespace rwkv;

extern "C" {

int rwkv_hip_copy_rows(rwkv_stream_t s, int tensors, void* const* dst_host, const void* const* src_host, const int64_t* planes_host,
                       const int64_t* row_bytes_host, int dst_rows, int src_rows, int n, const int32_t* to_host, const int32_t* from_host) {
  try {
    return copy_rows_launch(as_stream(s), tensors, dst_host, src_host, planes_host, row_bytes_host, dst_rows, src_rows, n, to_host, from_host);
  } catch (const std::bad_alloc&) {
    set_error("copy_rows: out of host memory");
    return RWKV_E_NOMEM;
  }
}

}  // extern "C"
