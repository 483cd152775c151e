// One token per row of logits, drawn with a given random number under the row's own temperature, top-k, top-p and min-p.  The
// reference's sampler (src/utils/sampling.cu:205-471) has one set of options for a batch, a generator of its own and no min-p.
//
//   z = fp32(logit) - penalty, rounded to fp32;  m = max z;  e_i = 2^((z_i - m) log2(e) / T), 0 below 2^-1000
//   order: larger z first, equal ones by index.  n_k = top_k;  n_p = least n whose first n entries hold top_p of the sum of e;
//   n_m = entries with e >= min_p;  kept = the first max(1, min(n_k, n_p, n_m)) entries, K = their sum
//   token = the first kept entry, by index, up to which the kept entries' sum is above u K
//   its log probability = -ln(1 + (K - e_token) / e_token), the difference summed without the token: nothing cancels
//
// Powers and sums are in 64 bits: which token is drawn goes by a comparison of two sums, and with fp32's 1e-7 one draw in some hundred
// of a row with many candidates would come out next to the one that the definition gives.  (The fp64 vector rate of this chip is that
// of fp32; an entry costs some twenty operations.)
//
// Three launches.  draw_stats_kernel reads the rows with the whole chip: per 64 entries (a slot) the largest z and, where the
// sum over the whole row is asked for, the sum of the slot's powers.  draw_pick_kernel has a block per row: the slots bound how small a kept
// entry can be, the slots that reach the bound are read again, and the entries above it go to a list in LDS, in order.  Lists are
// short for the filters that servers use; a row without filters needs none: its slots' sums give the token's slot.  draw_wide_kernel takes the
// rows whose list would overflow (flat rows with top-p alone, a large top-k, many equal logits), a block each with the whole row in registers.
#include <cfloat>
#include <climits>
#include <type_traits>

#include "ops.h"

namespace rwkv {

namespace {

constexpr int kSlot = 64;
constexpr int kStatsThreads = 256;
constexpr int kPickThreads = 1024;
constexpr int kWideThreads = 1024;
constexpr int kPickList = 4096;  // entries
constexpr int kWideList = 8192;
constexpr int kBuckets = 256;    // of a histogram
constexpr int kLast = 64;        // entries that one wavefront puts in order
constexpr int kWaveSlots = 256;  // slots of a wavefront that reach the bound
constexpr int kHeld = 8;         // of these, those whose entries it keeps in registers
constexpr int kMost = 256;       // of a block: a list of more slots takes longer to make than the search for a window
constexpr int kChunk = 64;       // slots of a wavefront in find_window: one entry of each a lane
constexpr int kWindow = kWideList * 3 / 4;  // entries that find_window narrows a row down to
constexpr double kLog2eD = 1.44269504088896340736;
constexpr double kLowestPower = -1000.0;  // octaves
constexpr double kWidest = 64.0;          // octaves that the first histogram covers

// What draw_pick_kernel hands on of a row with more candidates than its list holds
struct WideRow {
  double mass;            // what top_p holds; +infinity: no top_p
  float m;
  float lowest, highest;  // powers: no candidate lies below, and the cut not above
  int waits;
};

struct DrawArgs {
  const void* logits;
  int64_t ld;
  int V, slots, logit_rows;
  const int* source;
  const float* temperature;
  const int* top_k;
  const float* top_p;
  const float* min_p;
  const float* uniform;
  const float* penalties;  // [rows,V]
  int* token;
  float* logprob;
  double* slot_sum;  // [rows,slots]
  float* slot_max;   // [rows,slots]
  WideRow* wide;     // [rows]
};

// a value that every lane holds, in scalar registers
__device__ __forceinline__ float scalar(float v) { return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, v))); }
__device__ __forceinline__ int scalar(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ double scalar(double v) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<int>(b)), hi = __builtin_amdgcn_readfirstlane(static_cast<int>(b >> 32));
  return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}

// What a row asks for.  Filters that are off: top_k = INT_MAX, top_p >= 1, min_p <= 0.
struct Wish {
  double octaves;  // log2(e) / temperature
  double top_p, min_p, u;
  int top_k, source;
  bool valid, greedy;
  __device__ __forceinline__ bool free() const { return top_k == INT_MAX && top_p >= 1.0 && min_p <= 0.0; }
  __device__ __forceinline__ bool likely(double e) const { return !(min_p > 0.0) || e >= min_p; }
  __device__ __forceinline__ bool needs_sum() const { return !greedy && (top_p < 1.0 || free()); }
};
__device__ __forceinline__ Wish wish_of(const DrawArgs& a, int row) {
  Wish w;
  const float t = a.temperature ? a.temperature[row] : 1.0f;
  w.source = a.source ? a.source[row] : row;
  w.top_k = a.top_k ? a.top_k[row] : 0;
  if (w.top_k <= 0 || w.top_k >= a.V) w.top_k = INT_MAX;
  w.top_p = a.top_p ? a.top_p[row] : 1.0f;
  w.min_p = a.min_p ? fminf(a.min_p[row], 1.0f) : 0.0f;
  const float min_p = a.min_p ? a.min_p[row] : 0.0f;
  w.u = a.uniform[row];
  w.valid = w.source >= 0 && w.source < a.logit_rows && t >= 0.0f && w.top_p == w.top_p && min_p == min_p && w.u >= 0.0 && w.u <= 1.0;
  w.greedy = t == 0.0f;
  w.octaves = scalar(w.greedy ? 0.0 : kLog2eD / static_cast<double>(t));
  w.top_p = scalar(w.top_p);
  w.min_p = scalar(w.min_p);
  w.u = scalar(w.u);
  return w;
}

// a b + c with c in scalar registers (left to itself, the compiler moves every coefficient of a polynomial to the register of the sum first:
// half as many instructions again)
__device__ __forceinline__ double fma_scalar(double a, double b, double c) {
  double r;
  asm("v_fma_f64 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "s"(c));
  return r;
}
// e of an entry z <= m; 0 for -infinity.  2^f for |f| <= 1/2 is 1 + f q(f), exact at 0, with the polynomial through (2^f - 1) / f at the nine
// Chebyshev nodes of that range: 3.7e-14 off at most.
__device__ __forceinline__ double weight(float z, float m, double octaves) {
  const double y = (static_cast<double>(z) - static_cast<double>(m)) * octaves;
  const double n = rint(y);
  const double f = y - n;
  double q = fma_scalar(f, 1.0203121063391729e-07, 1.3255224878668817e-06);
  q = fma_scalar(q, f, 1.525268684626772e-05);
  q = fma_scalar(q, f, 0.00015403455852453838);
  q = fma_scalar(q, f, 0.0013333558179043112);
  q = fma_scalar(q, f, 0.009618129159402558);
  q = fma_scalar(q, f, 0.055504108664760424);
  q = fma_scalar(q, f, 0.2402265069581299);
  q = fma_scalar(q, f, 0.6931471805599453);
  const double v = ldexp(fma(q, f, 1.0), static_cast<int>(n));
  return y >= kLowestPower ? v : 0.0;  // (infinity times no octaves at all is a NaN, and none either)
}

template <int D>
__device__ __forceinline__ double lane_xor_d(double v) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = static_cast<uint32_t>(lane_xor_dpp<D>(static_cast<int>(b)));
  const uint32_t hi = static_cast<uint32_t>(lane_xor_dpp<D>(static_cast<int>(b >> 32)));
  return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}
__device__ __forceinline__ double row16_sum_d(double v) {
  v += lane_xor_d<8>(v);
  v += lane_xor_d<4>(v);
  v += lane_xor_d<2>(v);
  v += lane_xor_d<1>(v);
  return v;
}
__device__ __forceinline__ double wave_sum_d(double v) {
  v += lane_xor_d<32>(v);
  v += lane_xor_d<16>(v);
  return row16_sum_d(v);
}
template <typename T>
__device__ __forceinline__ T wave_upto(T v) {  // sum over this lane and those in front of it
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const T n = __shfl_up(v, off, 64);
    if (lane >= off) v += n;
  }
  return v;
}

// of up to 64 entries in order, one a lane: how many of the n are ahead of the lane's, and their sum
__device__ __forceinline__ void rank_of(float z, double e, int n, int& rank, double& ahead) {
  const int lane = threadIdx.x & 63;
  const uint64_t bits = __builtin_bit_cast(uint64_t, e);
  for (int j = 0; j < n; ++j) {
    const float zj = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, z), j));
    const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(bits), j), hi = __builtin_amdgcn_readlane(static_cast<int>(bits >> 32), j);
    const bool first = zj > z || (zj == z && j < lane);
    rank += first;
    ahead += first ? __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo) : 0.0;
  }
}

template <typename T>
struct Row {
  const T* logits;
  const float* penalties;
  int V;
  // (offsets of 32 bits from scalar addresses: a row is at most 4 MB)
  __device__ __forceinline__ float logit(uint32_t i) const {
    return static_cast<float>(*reinterpret_cast<const T*>(reinterpret_cast<const char*>(logits) + i * static_cast<uint32_t>(sizeof(T))));
  }
  __device__ __forceinline__ float penalty(uint32_t i) const {
    return *reinterpret_cast<const float*>(reinterpret_cast<const char*>(penalties) + i * 4u);
  }
  // entry i, or -infinity behind the end
  __device__ __forceinline__ float at(int i) const {
    if (i >= V) return -INFINITY;
    const float z = logit(i);
    return penalties ? z - penalty(i) : z;
  }
  // entries i, i + kSlot, ... to z[at], z[at + 1], ...: the row's last one in place of those behind it
  template <int N, int M>
  __device__ __forceinline__ void load(int i, float (&z)[M], int at) const {
#pragma unroll
    for (int k = 0; k < N; ++k) z[at + k] = logit(min(i + k * kSlot, V - 1));
    if (penalties) {
#pragma unroll
      for (int k = 0; k < N; ++k) z[at + k] -= penalty(min(i + k * kSlot, V - 1));
    }
  }
};
template <typename T>
__device__ __forceinline__ Row<T> row_of(const DrawArgs& a, int row, int source) {
  return {static_cast<const T*>(a.logits) + source * a.ld, a.penalties ? a.penalties + static_cast<int64_t>(row) * a.V : nullptr, a.V};
}

// f(z, i) for the entries of a run of slots, one of each to a lane: -infinity from `end` on.  The next eight are requested before the last
// ones are looked at.
template <typename T, typename F>
__device__ __forceinline__ void each_entry(const Row<T>& r, int first_slot, int end_slot, F&& f) {
  constexpr int kAhead = 8;
  const int end = min(end_slot * kSlot, r.V);
  float next[kAhead];
  int i = first_slot * kSlot + (threadIdx.x & 63);
  r.template load<kAhead>(i, next, 0);
  for (; i < end_slot * kSlot; i += kAhead * kSlot) {
    float z[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) z[k] = i + k * kSlot < end ? next[k] : -INFINITY;
    r.template load<kAhead>(i + kAhead * kSlot, next, 0);
#pragma unroll
    for (int k = 0; k < kAhead; ++k) f(z[k], i + k * kSlot);
  }
}

// A block takes kStatsThreads * 4 * NV entries of a row, 16 lanes a slot.  VEC: four entries are one aligned load.
template <typename T, bool VEC, int NV>
__global__ __launch_bounds__(kStatsThreads) void draw_stats_kernel(DrawArgs a) {
  typedef T vec_t __attribute__((ext_vector_type(4)));
  const int row = blockIdx.x;
  const Wish w = wish_of(a, row);
  if (!w.valid) return;
  const Row<T> r = row_of<T>(a, row, w.source);
  const bool sums = w.needs_sum();
  const int first = (blockIdx.y * kStatsThreads * NV + threadIdx.x) * 4;
  float z[NV][4];
#pragma unroll
  for (int q = 0; q < NV; ++q) {
    const int i = first + q * kStatsThreads * 4;
    if (VEC && i + 4 <= a.V) {
      const vec_t l = *reinterpret_cast<const vec_t*>(r.logits + i);
#pragma unroll
      for (int j = 0; j < 4; ++j) z[q][j] = static_cast<float>(l[j]);
      if (r.penalties) {
        const float4_t p = *reinterpret_cast<const float4_t*>(r.penalties + i);
#pragma unroll
        for (int j = 0; j < 4; ++j) z[q][j] -= p[j];
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) z[q][j] = r.at(i + j);
    }
  }
#pragma unroll
  for (int q = 0; q < NV; ++q) {
    const int slot = (first + q * kStatsThreads * 4) / kSlot;
    float m = -INFINITY;
#pragma unroll
    for (int j = 0; j < 4; ++j) m = fmaxf(m, z[q][j] < INFINITY ? z[q][j] : INFINITY);  // (a NaN counts as +infinity: no distribution)
    m = fmaxf(m, __builtin_bit_cast(float, lane_xor_dpp<8>(__builtin_bit_cast(int, m))));
    m = fmaxf(m, __builtin_bit_cast(float, lane_xor_dpp<4>(__builtin_bit_cast(int, m))));
    m = fmaxf(m, __builtin_bit_cast(float, lane_xor_dpp<2>(__builtin_bit_cast(int, m))));
    m = fmaxf(m, __builtin_bit_cast(float, lane_xor_dpp<1>(__builtin_bit_cast(int, m))));
    double sum = 0.0;
    if (sums) {
#pragma unroll
      for (int j = 0; j < 4; ++j) sum += weight(z[q][j], m, w.octaves);
      sum = row16_sum_d(sum);
    }
    if ((threadIdx.x & 15) == 0 && slot < a.slots) {
      const int64_t at = static_cast<int64_t>(row) * a.slots + slot;
      a.slot_max[at] = m;
      if (sums) a.slot_sum[at] = sum;
    }
  }
}

// What one wavefront or thread finds for its block, and what wavefronts exchange: by the block functions, and at places of their own
template <int NW, int LIST>
struct Shared {
  static constexpr int kWaves = NW, kList = LIST;
  double d[NW], d2[NW], total[NW], chunk[NW];
  float f[NW], f2[NW], most[NW], least[NW];
  int i[NW], reach[NW], entries[NW], counted[2][NW];
  float summed[2][NW];
  unsigned count[kBuckets];
  unsigned long long mass[kBuckets];
  float last_z[kLast];
  int last_i[kLast];
  alignas(8) float list_z[LIST];  // entries in order of their indexes
  int list_i[LIST];
  int bucket, missed, bucket_count, at, slot;
  double above_mass, before;
  float cut_z;
  int cut_i;
};

template <int NW>
__device__ __forceinline__ int block_min(int v, int (&buf)[NW]) {
  v = wave_reduce_dpp(v, [](int x, int y) { return min(x, y); });
  __syncthreads();
  if ((threadIdx.x & 63) == 0) buf[threadIdx.x >> 6] = v;
  __syncthreads();
  int r = buf[0];
#pragma unroll
  for (int i = 1; i < NW; ++i) r = min(r, buf[i]);
  return r;
}
template <int NW>
__device__ __forceinline__ double block_sum_d(double v, double (&buf)[NW]) {
  v = wave_sum_d(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) buf[threadIdx.x >> 6] = v;
  __syncthreads();
  double r = 0.0;
#pragma unroll
  for (int i = 0; i < NW; ++i) r += buf[i];
  return r;
}
// sum over the threads in front of this one, and over all
template <typename T, int NW>
__device__ __forceinline__ T block_before(T v, T (&buf)[NW], T* total) {
  const T upto = wave_upto(v);
  T before = __shfl_up(upto, 1, 64);
  if ((threadIdx.x & 63) == 0) before = T(0);
  __syncthreads();
  if ((threadIdx.x & 63) == 63) buf[threadIdx.x >> 6] = upto;
  __syncthreads();
  T base = T(0), all = T(0);
#pragma unroll
  for (int i = 0; i < NW; ++i) {
    if (i == static_cast<int>(threadIdx.x >> 6)) base = all;
    all += buf[i];
  }
  *total = all;
  return base + before;
}

// Buckets of equal width in z, from `top` down: a smaller z is never in an earlier bucket.
struct Buckets {
  double top, per_unit;
  __device__ __forceinline__ int of(float z) const {
    return static_cast<int>(fmin((top - static_cast<double>(z)) * per_unit, static_cast<double>(kBuckets - 1)));
  }
};
__device__ __forceinline__ Buckets buckets_of(double top, double range) { return {top, scalar(range > 0.0 ? kBuckets / range : 0.0)}; }

// What ends the kept entries, in the order: the first entry with which they are top_k or hold top_p
struct Cut {
  int top_k;
  double mass;  // +infinity: no top_p
  __device__ __forceinline__ bool open() const { return top_k == INT_MAX && !(mass < INFINITY); }
  __device__ __forceinline__ bool reached(int64_t n, double held) const { return n >= top_k || held >= mass; }
};

struct Found {
  float z;
  int i;  // kept: z above, or equal and no later index
  __device__ __forceinline__ bool keeps(float zi, int ii) const { return zi > z || (zi == z && ii <= i); }
};

// Entries in front of those that are looked at, in the order, and their sum; the ends of those
struct Span {
  int above;
  double above_mass;
  float low, high;
  __device__ __forceinline__ bool has(float z) const { return z >= low && z <= high; }
};

// One wavefront over a histogram: the first bucket in which the cut lies, the entries and the mass in front of it.  Where the sums do not
// reach the cut: kBuckets, or the last bucket that holds anything (`inside`: the cut is known to lie in this histogram, and rounding hides it).
template <typename S>
__device__ __forceinline__ void find_bucket(S& sh, const Cut& cut, int above, double above_mass, double unit, bool inside) {
  constexpr int kPer = kBuckets / 64;
  const int lane = threadIdx.x & 63;
  int n = 0;
  double held = 0.0;
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    n += sh.count[lane * kPer + j];
    held += static_cast<double>(sh.mass[lane * kPer + j]) * unit;
  }
  const int n_upto = wave_upto(n);
  const double held_upto = wave_upto(held);
  double held_before = __shfl_up(held_upto, 1, 64);
  if (lane == 0) held_before = 0.0;
  const uint64_t has = __ballot(n > 0), hit = __ballot(n > 0 && cut.reached(above + n_upto, above_mass + held_upto));
  if (hit == 0 && !inside) {
    if (lane == 0) sh.bucket = kBuckets;
    return;
  }
  const int owner = hit ? __ffsll(static_cast<unsigned long long>(hit)) - 1 : 63 - __clzll(static_cast<long long>(has));
  if (lane != owner) return;
  int at_n = above + n_upto - n;
  double at_held = above_mass + held_before;
  bool found = false;
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const int count = static_cast<int>(sh.count[lane * kPer + j]);
    if (count == 0 || found) continue;
    sh.bucket = lane * kPer + j;
    sh.bucket_count = count;
    sh.at = at_n;
    sh.above_mass = at_held;
    at_n += count;
    at_held += static_cast<double>(sh.mass[lane * kPer + j]) * unit;
    found = cut.reached(at_n, at_held);
  }
}

// Of `n` equal entries of weight e, how many the cut leaves
__device__ __forceinline__ int equal_ones(const Cut& cut, int above, double above_mass, int n, double e) {
  int64_t k = n;
  if (cut.top_k != INT_MAX) k = min(k, static_cast<int64_t>(cut.top_k) - above);
  if (cut.mass < INFINITY && e > 0.0) {
    int64_t p = static_cast<int64_t>(fmin(fmax(ceil((cut.mass - above_mass) / e), 1.0), static_cast<double>(n)));
    while (p > 1 && above_mass + static_cast<double>(p - 1) * e >= cut.mass) --p;
    while (p < n && above_mass + static_cast<double>(p) * e < cut.mass) ++p;
    k = min(k, p);
  }
  return static_cast<int>(max(k, static_cast<int64_t>(1)));
}

// The last entry that the cut leaves, among the entries of a span: the first `n` of the list, or, with a Row, all of a row until the list
// holds what is left.  Histograms of the span, each over the bucket of the one before in which the cut lies, until it holds few entries or
// equal ones.  False: the cut lies behind the span (`inside`: it is known not to).  Sums in fixed point: any order of the additions gives
// the same.
template <typename S, typename R>
__device__ __forceinline__ bool find_cut(S& sh, const R* row, int c0, int c1, int n, const Cut& cut, float m, double octaves, int V, Span span,
                                         Buckets buckets, bool inside, Found& found) {
  constexpr int kThreads = S::kWaves * 64;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int scale = 62 - (32 - __clz(V));  // (V weights of at most 1 stay below 2^63)
  const double unit = ldexp(1.0, -scale), per_unit = ldexp(1.0, scale);
  bool in_list = row == nullptr;
  const auto each = [&](auto&& f) {
    if (in_list) {
      for (int k = tid; k < n; k += kThreads) {
        const float z = sh.list_z[k];
        if (span.has(z)) f(z);
      }
    } else {
      each_entry(*row, c0, c1, [&](float z, int) {
        if (span.has(z)) f(z);
      });
    }
  };
  for (;; inside = true) {
    __syncthreads();
    for (int b = tid; b < kBuckets; b += kThreads) {
      sh.count[b] = 0;
      sh.mass[b] = 0;
    }
    __syncthreads();
    each([&](float z) {
      const int b = buckets.of(z);
      atomicAdd(&sh.count[b], 1u);
      if (cut.mass < INFINITY) atomicAdd(&sh.mass[b], static_cast<unsigned long long>(fma(weight(z, m, octaves), per_unit, 0.5)));
    });
    __syncthreads();
    if (wave == 0) find_bucket(sh, cut, span.above, span.above_mass, unit, inside);
    __syncthreads();
    const int b = scalar(sh.bucket);
    if (b == kBuckets) return false;
    const int count = scalar(sh.bucket_count);
    span.above = scalar(sh.at);
    span.above_mass = scalar(sh.above_mass);
    // the bucket's own ends
    float least = INFINITY, most = -INFINITY;
    each([&](float z) {
      if (buckets.of(z) == b) {
        least = fminf(least, z);
        most = fmaxf(most, z);
      }
    });
    least = wave_reduce_dpp(least, [](float x, float y) { return fminf(x, y); });
    most = wave_reduce_dpp(most, [](float x, float y) { return fmaxf(x, y); });
    if (lane == 0) {
      sh.f[wave] = least;
      sh.f2[wave] = most;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < S::kWaves; ++i) {
      least = fminf(least, sh.f[i]);
      most = fmaxf(most, sh.f2[i]);
    }
    span.low = scalar(least);
    span.high = scalar(most);
    const bool equal = span.low == span.high, last = equal || count <= kLast;
    if (last || (!in_list && count <= S::kList)) {
      // in order of their indexes: equal ones are counted, a few go to one wavefront, and those of a row that fit it to the list
      const int want = equal ? equal_ones(cut, span.above, span.above_mass, count, weight(span.low, m, octaves)) : 0;
      const int q = (n + kThreads - 1) / kThreads, k0 = min(tid * q, n), k1 = min(k0 + q, n);
      int have = 0, sum;
      if (in_list) {
        for (int k = k0; k < k1; ++k) have += span.has(sh.list_z[k]);
      } else {
        each_entry(*row, c0, c1, [&](float z, int) { have += __popcll(__ballot(span.has(z))); });
        if (lane != 0) have = 0;
      }
      int place = block_before(have, sh.i, &sum);
      const auto take = [&](float z, int i, int at) {
        if (equal) {
          if (at == want - 1) {
            sh.cut_z = z;
            sh.cut_i = i;
          }
        } else if (last) {
          if (at < kLast) {
            sh.last_z[at] = z;
            sh.last_i[at] = i;
          }
        } else if (at < S::kList) {
          sh.list_z[at] = z;
          sh.list_i[at] = i;
        }
      };
      if (in_list) {
        for (int k = k0; k < k1; ++k)
          if (span.has(sh.list_z[k])) take(sh.list_z[k], sh.list_i[k], place++);
      } else {
        place = scalar(place);
        each_entry(*row, c0, c1, [&](float z, int i) {
          const uint64_t hit = __ballot(span.has(z));
          if (hit >> lane & 1) take(z, i, place + __popcll(hit & ((1ull << lane) - 1)));
          place += __popcll(hit);
        });
      }
      __syncthreads();
      if (last) {
        if (!equal && wave == 0) {
          const float z = lane < count ? sh.last_z[lane] : -INFINITY;
          const double e = weight(z, m, octaves);
          int rank = 0;
          double ahead = 0.0;
          rank_of(z, e, count, rank, ahead);
          const bool hit = lane < count && cut.reached(static_cast<int64_t>(span.above) + rank + 1, span.above_mass + ahead + e);
          const int end = wave_reduce_dpp(hit ? rank : count - 1, [](int x, int y) { return min(x, y); });
          if (lane < count && rank == end) {
            sh.cut_z = z;
            sh.cut_i = sh.last_i[lane];
          }
        }
        __syncthreads();
        found = {scalar(sh.cut_z), scalar(sh.cut_i)};
        return true;
      }
      in_list = true;
      n = count;
    }
    buckets = buckets_of(span.high, static_cast<double>(span.high) - static_cast<double>(span.low));
  }
}

// One wavefront: the entry of a slot, given the sum in front of the slot and that of the kept entries in other slots
template <typename Weight, typename R, typename Answer>
__device__ __forceinline__ void draw_entry(Weight&& kept_weight, const R& r, int slot, double before, double target, double others, Answer&& answer) {
  const int lane = threadIdx.x & 63;
  const int i = slot * kSlot + lane;
  const double e = kept_weight(r.at(i), i);
  const double upto = before + wave_upto(e);
  const uint64_t has = __ballot(e > 0.0), hit = __ballot(e > 0.0 && upto > target);
  const int at = hit ? __ffsll(static_cast<unsigned long long>(hit)) - 1 : 63 - __clzll(static_cast<long long>(has));
  others += wave_sum_d(lane == at ? 0.0 : e);
  if (lane == at) answer(i, static_cast<float>(-log1p(others / e)));
}

// One wavefront over a list of up to 64 entries, in order: what is kept of them, and the token
template <typename S, typename Answer>
__device__ __forceinline__ void draw_from_few(const S& sh, int n, const Wish& w, const Cut& cut, float m, Answer&& answer) {
  const int lane = threadIdx.x & 63;
  const float z = lane < n ? sh.list_z[lane] : -INFINITY;
  const int i = lane < n ? sh.list_i[lane] : 0;
  const double e = weight(z, m, w.octaves);
  bool kept = lane < n;
  if (!cut.open()) {
    int rank = 0;
    double ahead = 0.0;
    rank_of(z, e, n, rank, ahead);
    const bool hit = kept && cut.reached(rank + 1, ahead + e);
    const int end = wave_reduce_dpp(hit ? rank : n, [](int x, int y) { return min(x, y); });
    kept = kept && rank <= end;
  }
  const double share = kept && w.likely(e) ? e : 0.0;
  const double upto = wave_upto(share);
  const double target = w.u * __shfl(upto, 63, 64);
  const uint64_t has = __ballot(share > 0.0), hit = __ballot(share > 0.0 && upto > target);
  const int at = hit ? __ffsll(static_cast<unsigned long long>(hit)) - 1 : 63 - __clzll(static_cast<long long>(has));
  const double others = wave_sum_d(lane == at ? 0.0 : share);
  if (lane == at) answer(i, static_cast<float>(-log1p(others / e)));
}

// A block over a list of n entries, in order, of which `found` and min_p keep some (the largest among them)
template <typename S, typename Answer>
__device__ __forceinline__ void draw_from_list(S& sh, int n, const Wish& w, const Found& found, float m, Answer&& answer) {
  constexpr int kThreads = S::kWaves * 64, kMine = S::kList / kThreads;  // a thread has so many neighbours
  const int tid = threadIdx.x;
  const int q = (n + kThreads - 1) / kThreads;
  double e[kMine], mine = 0.0;
#pragma unroll
  for (int j = 0; j < kMine; ++j) {
    e[j] = 0.0;
    const int k = tid * q + j;
    if (j < q && k < n) {
      const float z = sh.list_z[k];
      const double v = weight(z, m, w.octaves);
      if (found.keeps(z, sh.list_i[k]) && w.likely(v)) e[j] = v;
    }
    mine += e[j];
  }
  double kept;
  const double before = block_before(mine, sh.d, &kept);
  const double target = w.u * kept;
  int owner = block_min(mine > 0.0 && before + mine > target ? tid : INT_MAX, sh.i);
  if (owner == INT_MAX) owner = -block_min(mine > 0.0 ? -tid : 0, sh.i);
  if (tid == owner) {
    double upto = before;
    int pick = -1, last = 0;
#pragma unroll
    for (int j = 0; j < kMine; ++j) {
      upto += e[j];
      if (e[j] > 0.0) {
        last = j;
        if (pick < 0 && upto > target) pick = j;
      }
    }
    if (pick < 0) pick = last;
    sh.at = tid * q + pick;
  }
  __syncthreads();
  const int at = sh.at;
  double others = 0.0;
#pragma unroll
  for (int j = 0; j < kMine; ++j)
    if (tid * q + j != at || j >= q) others += e[j];
  others = block_sum_d(others, sh.d2);
  if (tid == 0) answer(sh.list_i[at], static_cast<float>(-log1p(others / weight(sh.list_z[at], m, w.octaves))));
}

constexpr int kPickWaves = kPickThreads / 64;
struct PickShared : Shared<kPickWaves, kPickList> {
  uint16_t slots[kPickWaves][kWaveSlots];
};

template <typename T>
__global__ __launch_bounds__(kPickThreads) void draw_pick_kernel(DrawArgs a) {
  __shared__ PickShared sh;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int row = blockIdx.x;
  const Wish w = wish_of(a, row);
  const auto fmax_op = [](float x, float y) { return fmaxf(x, y); };
  const auto fmin_op = [](float x, float y) { return fminf(x, y); };
  const auto answer = [&](int token, float logprob) {
    a.token[row] = token;
    if (a.logprob) a.logprob[row] = logprob;
  };
  if (tid == 0) a.wide[row].waits = 0;
  const float* slot_max = a.slot_max + static_cast<int64_t>(row) * a.slots;
  const double* slot_sum = a.slot_sum + static_cast<int64_t>(row) * a.slots;
  // a thread has neighbouring slots
  const int per = (a.slots + kPickThreads - 1) / kPickThreads;
  const int s0 = min(tid * per, a.slots), s1 = min(s0 + per, a.slots);
  float m = -INFINITY, lowest = INFINITY;
  if (w.valid)
    for (int s = s0; s < s1; ++s) {
      const float v = slot_max[s];
      m = fmaxf(m, v);
      if (v > -INFINITY) lowest = fminf(lowest, v);
    }
  m = wave_reduce_dpp(m, fmax_op);
  lowest = wave_reduce_dpp(lowest, fmin_op);
  if (lane == 0) {
    sh.most[wave] = m;
    sh.least[wave] = lowest;
  }
  for (int b = tid; b < kBuckets; b += kPickThreads) {
    sh.count[b] = 0;
    sh.mass[b] = 0;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kPickWaves; ++i) {
    m = fmaxf(m, sh.most[i]);
    lowest = fminf(lowest, sh.least[i]);
  }
  m = scalar(m);
  lowest = scalar(lowest);
  if (!(m > -INFINITY && m < INFINITY)) {
    if (tid == 0) answer(-1, 0.0f);
    return;
  }
  const Row<T> r = row_of<T>(a, row, w.source);

  if (w.greedy) {
    int s = INT_MAX;
    for (int k = s1 - 1; k >= s0; --k)
      if (slot_max[k] == m) s = k;
    s = block_min(s, sh.i);
    if (wave == 0) {
      const uint64_t hit = __ballot(r.at(s * kSlot + lane) == m);
      if (lane == 0) answer(s * kSlot + __ffsll(static_cast<unsigned long long>(hit)) - 1, 0.0f);
    }
    return;
  }

  const auto slot_share = [&](int s) { return slot_sum[s] * weight(slot_max[s], m, w.octaves); };
  double mine = 0.0;

  if (w.free()) {
    // by the slots' sums the slot, then its entry
    for (int s = s0; s < s1; ++s) mine += slot_share(s);
    double kept;
    const double before = block_before(mine, sh.d, &kept);
    const double target = w.u * kept;
    int owner = block_min(mine > 0.0 && before + mine > target ? tid : INT_MAX, sh.i);
    if (owner == INT_MAX) owner = -block_min(mine > 0.0 ? -tid : 0, sh.i);
    if (tid == owner) {
      double upto = before;
      bool sure = false;
      for (int s = s0; s < s1 && !sure; ++s) {
        const double e = slot_share(s);
        if (e > 0.0) {
          sh.slot = s;
          sh.before = upto;
          sure = upto + e > target;
        }
        upto += e;
      }
    }
    __syncthreads();
    const int slot = sh.slot;
    double others = 0.0;
    for (int s = s0; s < s1; ++s)
      if (s != slot) others += slot_share(s);
    others = block_sum_d(others, sh.d2);
    if (wave == 0) draw_entry([&](float z, int) { return weight(z, m, w.octaves); }, r, slot, sh.before, target, others, answer);
    return;
  }

  // how far down a kept entry can lie, from the slots
  const bool summed = w.needs_sum();
  double range = scalar(static_cast<double>(m) - static_cast<double>(lowest));
  if (range * w.octaves > kWidest) range = kWidest / w.octaves;
  const Buckets rough = buckets_of(m, scalar(range));
  constexpr double kUnit = 1.0 / (1ll << 40);  // (a row's sum is at most 2^20)
  for (int s = s0; s < s1; ++s) {
    const float v = slot_max[s];
    if (!(v > -INFINITY)) continue;
    const int b = rough.of(v);
    atomicAdd(&sh.count[b], 1u);
    if (summed) {
      const double share = slot_share(s);
      mine += share;
      atomicAdd(&sh.mass[b], static_cast<unsigned long long>(share * (1.0 / kUnit)));
    }
  }
  mine = wave_sum_d(mine);
  if (lane == 0) sh.total[wave] = mine;
  __syncthreads();
  double total = 0.0;
#pragma unroll
  for (int i = 0; i < kPickWaves; ++i) total += sh.total[i];
  total = scalar(total);
  const Cut cut = {w.top_k, scalar(w.top_p < 1.0 ? w.top_p * total : INFINITY)};
  const double width = scalar(range * w.octaves / kBuckets);  // octaves of a bucket
  const auto edge = [&](int b) { return __builtin_amdgcn_exp2f(static_cast<float>(-(b + 1) * width)); };  // the least power of a bucket
  if (wave == 0) {
    // Bucket b bounds the kept entries if, of the entries up to it, there are top_k (as many slots reach it), or top_p (what is in other
    // slots, and what their own entries below the bucket can hold at most, or all entries of the row, is less than the rest), or all that
    // min_p keeps.  It lies above
    // the cut if all entries of the slots that reach it are too few, and hold too little.
    constexpr int kPer = kBuckets / 64;
    const double spare = (1.0 - w.top_p) * total - 1e-8 * total;
    const double unlikely = w.min_p > 0.0 ? 1e-3 - __builtin_amdgcn_logf(static_cast<float>(w.min_p)) : INFINITY;
    int slots = 0;
    double held = 0.0;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      slots += sh.count[lane * kPer + j];
      held += static_cast<double>(sh.mass[lane * kPer + j]) * kUnit;
    }
    const int upto = wave_upto(slots);
    const double held_upto = wave_upto(held);
    int at = upto - slots;
    double at_held = held_upto - held;
    int bound = kBuckets - 1, missed = -1;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int b = lane * kPer + j;
      at += sh.count[b];
      at_held += static_cast<double>(sh.mass[b]) * kUnit;
      bool enough = at >= w.top_k || (b + 1) * width > unlikely;
      if (summed) enough |= fmin(total - at_held + static_cast<double>(at) * kSlot * edge(b) * 1.001, a.V * 1.001 * edge(b)) <= spare;
      if (enough) bound = min(bound, b);
      if (at < w.top_k / kSlot && (!summed || at_held < 0.999 * cut.mass)) missed = b;
    }
    bound = wave_reduce_dpp(bound, [](int x, int y) { return min(x, y); });
    missed = wave_reduce_dpp(missed, [](int x, int y) { return max(x, y); });
    if (lane == 0) {
      sh.bucket = bound;
      sh.missed = missed;
    }
  }
  __syncthreads();
  const int bound = scalar(sh.bucket);
  const auto candidate = [&](float z) { return z > -INFINITY && rough.of(z) <= bound; };

  // the slots that reach the bound, each wavefront its own, in order; the entries of the first ones are requested at once
  int reach = 0;
  for (int s = s0; s < s1; ++s) reach += candidate(slot_max[s]);
  const int reach_upto = wave_upto(reach);
  const int mine_reach = __builtin_amdgcn_readlane(reach_upto, 63);
  uint16_t* own = sh.slots[wave];
  for (int s = s0, to = reach_upto - reach; s < s1; ++s)
    if (candidate(slot_max[s])) {
      if (to < kWaveSlots) own[to] = static_cast<uint16_t>(s);
      ++to;
    }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  float held[kHeld];
#pragma unroll
  for (int k = 0; k < kHeld; ++k) held[k] = k < mine_reach ? r.at(own[k] * kSlot + lane) : -INFINITY;
  int entries = 0;
#pragma unroll
  for (int k = 0; k < kHeld; ++k) entries += __popcll(__ballot(candidate(held[k])));
  if (lane == 0) {
    sh.reach[wave] = mine_reach;
    sh.i[wave] = entries;
  }
  __syncthreads();
  int all = 0, widest = 0, n = 0, place = 0;
#pragma unroll
  for (int i = 0; i < kPickWaves; ++i) {
    all += sh.reach[i];
    widest = max(widest, sh.reach[i]);
    if (i == wave) place = n;
    n += sh.i[i];
  }
  bool fits = widest <= kWaveSlots && all <= kMost;
  if (fits && widest > kHeld) {
    for (int k = kHeld; k < mine_reach; ++k) entries += __popcll(__ballot(candidate(r.at(own[k] * kSlot + lane))));
    if (lane == 0) sh.entries[wave] = entries;
    __syncthreads();
    n = 0;
#pragma unroll
    for (int i = 0; i < kPickWaves; ++i) {
      if (i == wave) place = n;
      n += sh.entries[i];
    }
  }
  n = scalar(n);
  if (!fits || n > kPickList) {
    if (tid == 0)
      a.wide[row] = {cut.mass, m, bound < kBuckets - 1 ? edge(bound) * 0.999f : 0.0f, sh.missed >= 0 ? edge(sh.missed) * 1.001f : 1.0001f, 1};
    return;
  }
  const auto put = [&](float z, int slot) {
    const uint64_t hit = __ballot(candidate(z));
    if (hit >> lane & 1) {
      const int to = place + __popcll(hit & ((1ull << lane) - 1));
      sh.list_z[to] = z;
      sh.list_i[to] = slot * kSlot + lane;
    }
    place += __popcll(hit);
  };
#pragma unroll
  for (int k = 0; k < kHeld; ++k)
    if (k < mine_reach) put(held[k], own[k]);
  for (int k = kHeld; k < mine_reach; ++k) put(r.at(own[k] * kSlot + lane), own[k]);
  __syncthreads();
  if (n <= 64) {
    if (wave == 0) draw_from_few(sh, n, w, cut, m, answer);
    return;
  }
  Found found = {-INFINITY, INT_MAX};
  if (!cut.open()) {
    Buckets fine = rough;
    fine.per_unit *= kBuckets / (bound + 1.0);
    find_cut(sh, static_cast<const Row<T>*>(nullptr), 0, 0, n, cut, m, w.octaves, a.V, {0, 0.0, -FLT_MAX, FLT_MAX}, fine, false, found);
  }
  draw_from_list(sh, n, w, found, m, answer);
}

// ---- rows with more candidates than a list holds -----------------------------------------------------------------------
constexpr int kWideWaves = kWideThreads / 64;
struct WideShared : Shared<kWideWaves, kWideList> {
  float queue[kWideWaves][128];
};
static_assert(kMaxLogprobVocab / kSlot / kWideWaves <= kWideList / 2, "the sums of a chunk's slots lie where the list was");

struct WindowOut {
  Span span;
  int n;              // entries in the list
  int mine, mine_at;  // of them, this wavefront's
  double kept_above;  // and its kept entries above them, by lanes
};

enum class Window { kNone, kAll, kFound };

// For rows with many candidates: a window of values about the cut that fits the list.  Every thread keeps fp32 powers of its entries
// in registers, and the block halves the range of powers from `lowest` to `highest` by counting and summing, as long as fp32 tells on which
// side the cut lies.  What lies above the window is then counted and summed in 64 bits, and the window's entries go to the list, in order.
// (The caller finds out whether the cut lies inside.)  kAll: no candidate lies behind the cut.  kNone: nothing is found.
// Halving takes 4 to 7 steps between the bounds that the slots give, a straight line through the sums two more.
template <typename T>
__device__ __forceinline__ Window find_window(WideShared& sh, const Row<T>& r, int c0, int c1, const Wish& w, const Cut& cut, const WideRow& wide,
                                              WindowOut& out) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const float m = wide.m;
  const float octaves = fminf(static_cast<float>(w.octaves), 1e30f);
  const float mass = static_cast<float>(cut.mass);
  constexpr float kUnsure = 2e-5f;  // of a sum: the powers are good to 3e-6 down to 2^-64, and as many additions to as much
  const auto reached = [&](int n, float held) { return n >= cut.top_k || held >= mass * (1.0f + kUnsure); };
  const auto missed = [&](int n, float held) { return n < cut.top_k && held < mass * (1.0f - kUnsure); };
  uint32_t lo = __builtin_bit_cast(uint32_t, fmaxf(wide.lowest, 0x1p-120f)), hi = __builtin_bit_cast(uint32_t, wide.highest);
  if (lo >= hi) return Window::kAll;
  float x[kChunk];
  const int first = c0 * kSlot + lane, end = min(c1 * kSlot, r.V);
  constexpr int kAhead = 16;  // (more loads at once, and their addresses need the registers of the entries)
#pragma unroll
  for (int g = 0; g < kChunk; g += kAhead) {
    r.template load<kAhead>(first + g * kSlot, x, g);
#pragma unroll
    for (int k = g; k < g + kAhead; ++k) x[k] = first + k * kSlot < end ? __builtin_amdgcn_exp2f((x[k] - m) * octaves) : 0.0f;
    __builtin_amdgcn_sched_barrier(0);
  }
  // (one place in the code that counts, whatever for: unrolled over 64 registers it is 2 KB, and instructions that are executed once cost
  // their way from memory)
  const bool by_mass = cut.mass < INFINITY, by_count = cut.top_k != INT_MAX;
  enum { kLow, kHalve, kBelow, kAbove } state = kLow;
  constexpr uint32_t kNear = 1u << 15;  // 2^-8 of a value
  uint32_t at = lo, mid = 0, d = 0;
  int n_lo = 0, n_hi = 0, turn = 0;
  float held_lo = 0.0f, held_hi = 0.0f;
  // how many entries there can be between the two ends: none weighs less than the lower one
  const auto between = [&] {
    const float most = by_mass ? (held_lo - held_hi) / __builtin_bit_cast(float, lo) : INFINITY;
    return by_count ? fminf(most, static_cast<float>(n_lo - n_hi)) : most;
  };
  for (;;) {
    const float least = __builtin_bit_cast(float, at);
    int n = 0;
    float held = 0.0f;
    if (by_mass) {
#pragma unroll
      for (int k = 0; k < kChunk; ++k) held += x[k] >= least ? x[k] : 0.0f;
    }
    if (by_count) {
#pragma unroll
      for (int k = 0; k < kChunk; ++k) n += x[k] >= least;
    }
    held = wave_reduce_dpp(held, [](float x, float y) { return x + y; });
    n = wave_reduce_dpp(n, [](int x, int y) { return x + y; });
    // (two places in turn: a wavefront that writes one again has been past the barrier behind which the other was read)
    turn ^= 1;
    if (lane == 0) {
      sh.counted[turn][wave] = n;
      sh.summed[turn][wave] = held;
    }
    __syncthreads();
    n = 0;
    held = 0.0f;
#pragma unroll
    for (int i = 0; i < kWideWaves; ++i) {
      n += sh.counted[turn][i];
      held += sh.summed[turn][i];
    }
    n = scalar(n);
    held = scalar(held);
    const bool is_reached = reached(n, held), is_missed = missed(n, held);
    if (state == kLow) {
      if (is_missed) return Window::kAll;
      if (!is_reached) return Window::kNone;
      n_lo = n;
      held_lo = held;
      state = kHalve;
    } else if (state == kHalve) {
      if (is_reached) {
        lo = at;
        n_lo = n;
        held_lo = held;
      } else if (is_missed) {
        hi = at;
        n_hi = n;
        held_hi = held;
      } else {  // next to the cut: as close to it as fp32 can tell
        mid = at;
        d = kNear;
        state = kBelow;
      }
    } else if (state == kBelow) {
      if (is_reached) lo = at;
      d *= 4;
    } else {
      if (is_missed) hi = at;
      d *= 4;
    }
    if (state == kHalve) {
      if (between() <= kWindow || hi - lo <= 1) break;
      at = lo + (hi - lo) / 2;
    }
    if (state == kBelow) {
      if (mid - lo > d) {
        at = mid - d;
      } else {
        state = kAbove;
        d = kNear;
      }
    }
    if (state == kAbove) {
      if (hi - mid <= d) break;
      at = mid + d;
    }
  }
  // the window's ends as logits, further apart than fp32 powers are off
  constexpr float kApart = 1e-4f;  // octaves
  const float top = static_cast<float>(m + (__builtin_amdgcn_logf(__builtin_bit_cast(float, hi)) + kApart) / w.octaves);
  const float bottom = static_cast<float>(m + (__builtin_amdgcn_logf(__builtin_bit_cast(float, lo)) - kApart) / w.octaves);
  // What lies above the window is a fifth of a flat row's entries at a top_p of 0.95, spread evenly: it queues up until there is one for every
  // lane (a power takes as long for one lane as for 64).  The window's entries go to the list, each wavefront's to a part of its own.
  constexpr int kPart = kWideList / kWideWaves;
  double sum = 0.0, kept = 0.0;
  int higher = 0, inside = 0, waiting = 0;
  float least = INFINITY, most = -INFINITY;
  const bool picky = w.min_p > 0.0;
  const uint64_t in_front = (1ull << lane) - 1;
  float* queue = sh.queue[wave];
  const auto add = [&](float z) {
    const double v = weight(z, m, w.octaves);
    sum += v;
    if (picky) kept += v >= w.min_p ? v : 0.0;
  };
  each_entry(r, c0, c1, [&](float z, int i) {
    const uint64_t over = __ballot(z > top), in = __ballot(z >= bottom && z <= top && z > -INFINITY);
    if (over != 0) {
      if (over >> lane & 1) queue[waiting + __popcll(over & in_front)] = z;
      waiting += __popcll(over);
      if (waiting >= 64) {
        higher += 64;
        waiting -= 64;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        add(queue[lane]);
        const float next = queue[64 + lane];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        queue[lane] = next;
      }
    }
    if (in != 0) {
      const int to = inside + __popcll(in & in_front);
      if ((in >> lane & 1) && to < kPart) {
        sh.list_z[wave * kPart + to] = z;
        sh.list_i[wave * kPart + to] = i;
        least = fminf(least, z);
        most = fmaxf(most, z);
      }
      inside += __popcll(in);
    }
  });
  higher += waiting;
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  add(lane < waiting ? queue[lane] : -INFINITY);
  const double sum_mine = sum;
  sum = wave_sum_d(sum);
  least = wave_reduce_dpp(least, [](float x, float y) { return fminf(x, y); });
  most = wave_reduce_dpp(most, [](float x, float y) { return fmaxf(x, y); });
  __syncthreads();
  if (lane == 0) {
    sh.d[wave] = sum;
    sh.i[wave] = higher;
    sh.entries[wave] = inside;
    sh.f[wave] = least;
    sh.f2[wave] = most;
  }
  __syncthreads();
  int all = 0, place = 0, n = 0, widest = 0;
  sum = 0.0;
#pragma unroll
  for (int i = 0; i < kWideWaves; ++i) {
    if (i == wave) place = all;
    all += sh.entries[i];
    widest = max(widest, sh.entries[i]);
    n += sh.i[i];
    sum += sh.d[i];
    least = fminf(least, sh.f[i]);
    most = fmaxf(most, sh.f2[i]);
  }
  if (all == 0 || all > kWideList || widest > kPart || cut.reached(n, sum)) return Window::kNone;
  // the parts move together
  float z[kPart / 64];
  int i[kPart / 64];
#pragma unroll
  for (int k = 0; k < kPart / 64; ++k) {
    z[k] = sh.list_z[wave * kPart + k * 64 + lane];
    i[k] = sh.list_i[wave * kPart + k * 64 + lane];
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kPart / 64; ++k)
    if (k * 64 + lane < inside) {
      sh.list_z[place + k * 64 + lane] = z[k];
      sh.list_i[place + k * 64 + lane] = i[k];
    }
  out.span = {n, scalar(sum), scalar(least), scalar(most)};
  out.n = all;
  out.mine = inside;
  out.mine_at = place;
  out.kept_above = picky ? kept : sum_mine;
  __syncthreads();
  return Window::kFound;
}

template <typename T>
__global__ __launch_bounds__(kWideThreads) void draw_wide_kernel(DrawArgs a) {
  __shared__ WideShared sh;
  const int row = blockIdx.x;
  const WideRow wide = a.wide[row];
  if (!wide.waits) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const Wish w = wish_of(a, row);
  const float m = wide.m;
  const Cut cut = {w.top_k, wide.mass};
  const Row<T> r = row_of<T>(a, row, w.source);
  const auto answer = [&](int token, float logprob) {
    a.token[row] = token;
    if (a.logprob) a.logprob[row] = logprob;
  };
  const int chunk = (a.slots + kWideWaves - 1) / kWideWaves;  // slots of a wavefront
  const int c0 = min(wave * chunk, a.slots), c1 = min(c0 + chunk, a.slots);

  Found found = {-INFINITY, INT_MAX};
  WindowOut out;
  Window window = cut.open() ? Window::kAll : Window::kNone;
  if (!cut.open() && chunk <= kChunk && cut.mass > 0.0) {
    window = find_window(sh, r, c0, c1, w, cut, wide, out);
    if (window == Window::kFound &&
        !find_cut(sh, static_cast<const Row<T>*>(nullptr), 0, 0, out.n, cut, m, w.octaves, a.V, out.span,
                  buckets_of(out.span.high, static_cast<double>(out.span.high) - static_cast<double>(out.span.low)), false, found))
      window = Window::kNone;  // (beside the cut)
  }
  if (window == Window::kNone)
    find_cut(sh, &r, c0, c1, 0, cut, m, w.octaves, a.V, {0, 0.0, -FLT_MAX, FLT_MAX}, buckets_of(m, kWidest / w.octaves), false, found);

  // the kept entries' sums by wavefronts, of the entry's wavefront by slots, of its slot by entries
  const auto kept_weight = [&](float z, int i) {
    const double e = weight(z, m, w.octaves);
    return found.keeps(z, i) && w.likely(e) ? e : 0.0;
  };
  double share = 0.0;
  if (window == Window::kFound) {
    // (a list in order: this wavefront's part of it is what lies in its chunk)
    share = out.kept_above;
    for (int k = lane; k < out.mine; k += 64) share += kept_weight(sh.list_z[out.mine_at + k], sh.list_i[out.mine_at + k]);
  } else {
    each_entry(r, c0, c1, [&](float z, int i) { share += kept_weight(z, i); });
  }
  share = wave_sum_d(share);
  __syncthreads();
  if (lane == 0) sh.chunk[wave] = share;
  __syncthreads();
  double kept = 0.0;
#pragma unroll
  for (int i = 0; i < kWideWaves; ++i) kept += sh.chunk[i];
  const double target = w.u * kept;
  double upto = 0.0, before = 0.0, others = 0.0;
  int owner = -1;
  bool sure = false;
#pragma unroll
  for (int i = 0; i < kWideWaves; ++i) {
    const double v = sh.chunk[i];
    if (v > 0.0 && !sure) {
      owner = i;
      before = upto;
      sure = upto + v > target;
    }
    upto += v;
  }
#pragma unroll
  for (int i = 0; i < kWideWaves; ++i) others += i == owner ? 0.0 : sh.chunk[i];
  const int o0 = owner * chunk, slots = min(o0 + chunk, a.slots) - o0;
  double* sums = reinterpret_cast<double*>(sh.list_z);
  for (int s = wave; s < slots; s += 4 * kWideWaves) {
    float z[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) z[k] = s + k * kWideWaves < slots ? r.at((o0 + s + k * kWideWaves) * kSlot + lane) : -INFINITY;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const double sum = wave_sum_d(kept_weight(z[k], (o0 + s + k * kWideWaves) * kSlot + lane));
      if (lane == 0 && s + k * kWideWaves < slots) sums[s + k * kWideWaves] = sum;
    }
  }
  __syncthreads();
  if (wave != 0) return;
  // one wavefront over up to 1024 sums, 64 at a time
  int slot = 0;
  double slot_before = 0.0;
  sure = false;
  for (int s = 0; s < slots && !sure; s += 64) {
    const double own = s + lane < slots ? sums[s + lane] : 0.0;
    const double own_upto = before + wave_upto(own);
    const uint64_t has = __ballot(own > 0.0), hit = __ballot(own > 0.0 && own_upto > target);
    if (has != 0) {
      const int at = hit ? __ffsll(static_cast<unsigned long long>(hit)) - 1 : 63 - __clzll(static_cast<long long>(has));
      slot = s + at;
      slot_before = at == 0 ? before : __shfl(own_upto, at - 1, 64);
      sure = hit != 0;
    }
    before = __shfl(own_upto, 63, 64);
  }
  double rest = 0.0;
  for (int s = lane; s < slots; s += 64) rest += s == slot ? 0.0 : sums[s];
  draw_entry(kept_weight, r, o0 + slot, slot_before, target, others + wave_sum_d(rest), answer);
}

// What the penalties are after the token: all decayed, the token's own raised by `presence` where it had none, else by `frequency`.
__global__ __launch_bounds__(256) void draw_penalties_kernel(int V, const float* penalties, float* out, const int* token, const float* presence,
                                                             const float* frequency, const float* decay) {
  const int row = blockIdx.x;
  const int pick = token[row];
  const float keep = decay ? decay[row] : 1.0f;
  const float once = presence ? presence[row] : 0.0f, again = frequency ? frequency[row] : 0.0f;
  const int64_t base = static_cast<int64_t>(row) * V;
  for (int k = 0; k < 16; ++k) {
    const int i = (blockIdx.y * 16 + k) * 256 + threadIdx.x;
    if (i >= V) break;
    const float p = penalties[base + i];
    out[base + i] = fmaf(p, keep, i != pick ? 0.0f : p == 0.0f ? once : again);
  }
}

template <typename T>
void launch_draw(hipStream_t st, int rows, const DrawArgs& a, bool vec) {
  const auto stats = [&](auto aligned, auto vectors) {
    constexpr bool kVec = decltype(aligned)::value;
    constexpr int kNv = decltype(vectors)::value;
    hipLaunchKernelGGL((draw_stats_kernel<T, kVec, kNv>), dim3(rows, ceil_div(a.V, kStatsThreads * 4 * kNv)), dim3(kStatsThreads), 0, st, a);
  };
  const bool few = static_cast<int64_t>(rows) * ceil_div(a.V, 4096) < 1024;
  if (vec && few) stats(std::true_type{}, std::integral_constant<int, 1>{});
  else if (vec) stats(std::true_type{}, std::integral_constant<int, 4>{});
  else stats(std::false_type{}, std::integral_constant<int, 1>{});
  hipLaunchKernelGGL((draw_pick_kernel<T>), dim3(rows), dim3(kPickThreads), 0, st, a);
  if (a.top_k || a.top_p || a.min_p) hipLaunchKernelGGL((draw_wide_kernel<T>), dim3(rows), dim3(kWideThreads), 0, st, a);
}

size_t draw_bytes(int rows, int V) {
  const size_t slots = static_cast<size_t>(rows) * ceil_div(V, kSlot);
  return (slots * 12 + rows * sizeof(WideRow) + 15) / 16 * 16;
}

}  // namespace

}  // namespace rwkv

using namespace rwkv;

extern "C" {

int rwkv_hip_draw_tokens_workspace(int rows, int V, size_t* bytes) {
  RWKV_REQUIRE(bytes && rows > 0 && V > 0 && V <= kMaxLogprobVocab, "draw_tokens_workspace: bad arguments");
  *bytes = draw_bytes(rows, V);
  return RWKV_OK;
}

int rwkv_hip_draw_tokens(rwkv_stream_t s, int rows, int V, int io, const void* logits, int64_t ld, int logit_rows, const void* source,
                         const void* temperature, const void* top_k, const void* top_p, const void* min_p, const void* uniform,
                         const void* penalties, const void* presence, const void* frequency, const void* decay, void* penalties_out, void* token,
                         void* logprob, void* workspace, size_t workspace_bytes) {
  RWKV_REQUIRE(rows > 0 && logit_rows > 0, "draw_tokens: rows must be positive, got %d of %d", rows, logit_rows);
  RWKV_REQUIRE(V > 0 && V <= kMaxLogprobVocab, "draw_tokens: V must lie in 1 .. %d, got %d", kMaxLogprobVocab, V);
  RWKV_REQUIRE(io == RWKV_IO_F16 || io == RWKV_IO_F32, "draw_tokens: unknown element type %d", io);
  RWKV_REQUIRE(logits && uniform && token, "draw_tokens: NULL logits, uniform or token");
  RWKV_REQUIRE(ld >= V || logit_rows == 1, "draw_tokens: rows of %d entries lie %lld apart", V, static_cast<long long>(ld));
  RWKV_REQUIRE(source || logit_rows >= rows, "draw_tokens: %d rows of %d without their sources", rows, logit_rows);
  RWKV_REQUIRE((reinterpret_cast<uintptr_t>(logits) & (io == RWKV_IO_F16 ? 1 : 3)) == 0, "draw_tokens: misaligned logits");
  for (const void* p : {source, temperature, top_k, top_p, min_p, uniform, penalties, presence, frequency, decay, static_cast<const void*>(penalties_out),
                        static_cast<const void*>(token), static_cast<const void*>(logprob)})
    RWKV_REQUIRE((reinterpret_cast<uintptr_t>(p) & 3) == 0, "draw_tokens: 32-bit tensors must be aligned to 4 bytes");
  RWKV_REQUIRE(penalties || !(penalties_out || presence || frequency || decay), "draw_tokens: what becomes of penalties without any");
  RWKV_REQUIRE(penalties_out || !(presence || frequency || decay), "draw_tokens: presence, frequency and decay without penalties_out");
  const size_t need = draw_bytes(rows, V);
  RWKV_REQUIRE(workspace && workspace_bytes >= need && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0,
               "draw_tokens: workspace of %zu bytes (aligned to 16) needed, got %zu", need, workspace_bytes);
  const int slots = ceil_div(V, kSlot);
  double* sums = static_cast<double*>(workspace);
  WideRow* wide = reinterpret_cast<WideRow*>(sums + static_cast<size_t>(rows) * slots);
  const DrawArgs a = {logits, ld, V, slots, logit_rows, static_cast<const int*>(source), static_cast<const float*>(temperature),
                      static_cast<const int*>(top_k), static_cast<const float*>(top_p), static_cast<const float*>(min_p),
                      static_cast<const float*>(uniform), static_cast<const float*>(penalties), static_cast<int*>(token), static_cast<float*>(logprob),
                      sums, reinterpret_cast<float*>(wide + rows), wide};
  const uintptr_t misaligned = io == RWKV_IO_F16 ? 7 : 15;
  const bool vec = (reinterpret_cast<uintptr_t>(logits) & misaligned) == 0 && (ld % 4 == 0 || logit_rows == 1) &&
                   (!penalties || ((reinterpret_cast<uintptr_t>(penalties) & 15) == 0 && (V % 4 == 0 || rows == 1)));
  if (io == RWKV_IO_F16) launch_draw<half_t>(as_stream(s), rows, a, vec);
  else launch_draw<float>(as_stream(s), rows, a, vec);
  if (penalties_out)
    hipLaunchKernelGGL(draw_penalties_kernel, dim3(rows, ceil_div(V, 4096)), dim3(256), 0, as_stream(s), V, static_cast<const float*>(penalties),
                       static_cast<float*>(penalties_out), static_cast<const int*>(token), static_cast<const float*>(presence),
                       static_cast<const float*>(frequency), static_cast<const float*>(decay));
  RWKV_LAUNCH_CHECK();
  return RWKV_OK;
}

}  // extern "C"
