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
// of a row with many candidates would come out next to the one that the definition gives.  (An instruction on fp64 takes twice as long
// as one on fp32 here; an entry costs some thirty of both.)
//
// Two launches.  draw_stats_kernel reads the rows with the whole chip: per 64 entries (a slot) the largest z; per 4096 (a part), where the
// row asks for it, sums of powers and a histogram of them.  draw_pick_kernel has a block per row, which finds out how small a kept entry can be,
// reads the slots that reach that far again and puts their entries that do in a list in LDS, in order.  Lists are short for the filters that
// servers use.  Where the list would overflow (flat rows with top-p alone, a large top-k) it holds the entries about the cut only, the histograms
// say what lies above them, and a third look at one wavefront's share of the row finds the token.  Rows without filters need no list: the sums of
// their slots give the token's.
#include <algorithm>
#include <cfloat>
#include <climits>
#include <type_traits>

#include "ops.h"

namespace rwkv {

namespace {

constexpr int kSlot = 64;
constexpr int kPart = 4096;      // entries of a block of draw_stats_kernel
constexpr int kStatsThreads = 256;
constexpr int kPickThreads = 512;
constexpr int kList = 6144;      // entries
constexpr int kBuckets = 256;    // of a histogram
constexpr int kSums = kBuckets / 64;
constexpr int kLast = 64;        // entries that one wavefront puts in order
constexpr int kWaveSlots = 256;  // slots of a wavefront that reach the bound
constexpr int kHeld = 8;         // of these, those that it reads at once
// Slots of a block that reach the bound: with more of them the histograms of a row that has some lead to the cut sooner than a list of the
// entries.  V = 65536, list / window, us: 236 slots 26 / 31 at 8 rows and 47 / 54 at 256, 371 slots 31 / 31 and 52 / 55, 659 38 / 31 and 62 / 55.
constexpr int kMost = 384;
// A top_k up to which a row does without histograms, and the most slots to a place of it (the slots' maxima bound the kept entries the worse the
// fewer they are).  Without / with histograms, us: 8 rows of 65536, top_k 128 19 / 23, 512 29 / 31, 640 34 / 31; 256 rows 29 / 45, 42 / 55, 46 / 55;
// 8 rows of 16384 (256 slots), top_k 128 20 / 23, 192 24 / 24, 256 55 / 26; of 4096 (64 slots), 32 19 / 20, 64 28 / 24.
constexpr int kListed = 512;
constexpr int kSlotsListed = 2;
constexpr int kGrid = 8;         // buckets of the parts' histograms in an octave
constexpr double kOne = 2251799813685248.0;  // 2^51: 2^12 powers of at most 1 stay below 2^64
constexpr double kPartOne = kOne / 2.0;      // of the parts' histograms, where they are at most 2
constexpr double kLog2eD = 1.44269504088896340736, kLn2D = 0.69314718055994530942;
constexpr double kLowestPower = -1000.0;  // octaves
constexpr double kWidest = 64.0;          // octaves that the first histogram covers

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
  // What draw_stats_kernel leaves: the largest entry of every slot and part; for rows that need them the sums of the slots' powers, against
  // the part's largest entry, or the parts' histograms: powers (raised by part_raised, times kPartOne) and numbers of the entries, and the powers' sums
  // over 64 buckets (times kPartOne)
  int parts;
  double* slot_sum;               // [rows,slots]
  double* part_sum;               // [rows,parts,kSums]
  unsigned long long* part_mass;  // [rows,parts,kBuckets]
  float* slot_max;                // [rows,slots]
  float* part_max;                // [rows,parts]
  unsigned* part_count;           // [rows,parts,kBuckets]
};

// a value that every lane holds, in scalar registers
__device__ __forceinline__ float scalar(float v) { return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, v))); }
__device__ __forceinline__ int scalar(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ double scalar(double v) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<int>(b)), hi = __builtin_amdgcn_readfirstlane(static_cast<int>(b >> 32));
  return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}

// What makes powers of differences: log2(e) / temperature, the difference that 2^kLowestPower belongs to, and buckets of the grid to a unit
struct Power {
  double octaves, lowest;
  float grid;
};

// What a row asks for.  Filters that are off: top_k = INT_MAX, top_p >= 1, min_p <= 0.
struct Wish {
  Power power;
  double top_p, min_p, u;
  int top_k, listed, source;
  bool valid, greedy;
  __device__ __forceinline__ bool free() const { return top_k == INT_MAX && top_p >= 1.0 && min_p <= 0.0; }
  // a kept entry is the token once the sum up to it passes this (1: none but the last one, whatever the sums are rounded to)
  __device__ __forceinline__ double target(double kept) const { return u < 1.0 ? u * kept : INFINITY; }
  __device__ __forceinline__ bool likely(double e) const { return !(min_p > 0.0) || e >= min_p; }
  // (a list of top_k entries, and of the rest of their slots, is short)
  __device__ __forceinline__ bool needs_histogram() const { return !greedy && !free() && top_k > listed; }
  __device__ __forceinline__ bool needs_sums() const { return !greedy && (free() || (top_p < 1.0 && !needs_histogram())); }
};
__device__ __forceinline__ Wish wish_of(const DrawArgs& a, int row) {
  Wish w;
  const float t = a.temperature ? a.temperature[row] : 1.0f;
  w.source = a.source ? a.source[row] : row;
  w.top_k = a.top_k ? a.top_k[row] : 0;
  if (w.top_k <= 0 || w.top_k >= a.V) w.top_k = INT_MAX;
  w.listed = min(kListed, a.slots / kSlotsListed);
  w.top_p = a.top_p ? a.top_p[row] : 1.0f;
  w.min_p = a.min_p ? fminf(a.min_p[row], 1.0f) : 0.0f;
  const float min_p = a.min_p ? a.min_p[row] : 0.0f;
  w.u = a.uniform[row];
  w.valid = w.source >= 0 && w.source < a.logit_rows && t >= 0.0f && w.top_p == w.top_p && min_p == min_p && w.u >= 0.0 && w.u <= 1.0;
  w.greedy = t == 0.0f;
  w.power.octaves = scalar(w.greedy ? 0.0 : fmax(kLog2eD / static_cast<double>(t), kLowestPower / -1e300));  // (an infinite t: -1e300 is the lowest)
  w.power.lowest = scalar(fmax(kLowestPower * kLn2D * static_cast<double>(t), -1e300));  // (above -infinity at any temperature)
  w.power.grid = scalar(static_cast<float>(w.power.octaves * kGrid));
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
// e of an entry z <= m; 0 for -infinity.  The difference's octaves are rounded by the addition of a number whose last bit is 1, and the integer
// is what its low bits then hold.  2^f for |f| <= 1/2 is 1 + f q(f), exact at 0, with the polynomial through (2^f - 1) / f at the nine Chebyshev
// nodes of that range: 3.7e-14 off at most.  `raised`: octaves to multiply it by.  ALWAYS: 2^kLowestPower in place of 0 (for units in which that is
// nothing).
constexpr double kNinth = 1.0203121063391729e-07;  // the highest coefficient
constexpr double kRound = 6755399441055744.0;      // 1.5 2^52
template <bool ALWAYS = false>
__device__ __forceinline__ double weight(float z, float m, const Power& p, double ninth = kNinth, double round = kRound, int raised = 0) {
  double d = static_cast<double>(z) - static_cast<double>(m);
  if constexpr (ALWAYS) d = fmax(d, p.lowest);
  const double y = fma(d, p.octaves, round);
  const int n = static_cast<int>(static_cast<uint32_t>(__builtin_bit_cast(uint64_t, y)));
  const double f = fma(d, p.octaves, round - y);
  double q = fma_scalar(f, ninth, 1.3255224878668817e-06);
  q = fma_scalar(q, f, 1.525268684626772e-05);
  q = fma_scalar(q, f, 0.00015403455852453838);
  q = fma_scalar(q, f, 0.0013333558179043112);
  q = fma_scalar(q, f, 0.009618129159402558);
  q = fma_scalar(q, f, 0.055504108664760424);
  q = fma_scalar(q, f, 0.2402265069581299);
  q = fma_scalar(q, f, 0.6931471805599453);
  const double v = ldexp(fma(q, f, 1.0), n + raised);
  if constexpr (ALWAYS) return v;
  return d >= p.lowest ? v : 0.0;  // (not where d is -infinity or, with an m of -infinity, a NaN)
}
// A power in units of 1 / `one`, up to 2^51 of them or a little more: 2^52 + e one, rounded, holds it in its last 52 bits.
__device__ __forceinline__ unsigned long long in_units(double e, double one = kOne, double two = 2.0 * kOne) {
  return __builtin_bit_cast(unsigned long long, fma(e, one, two)) - 0x4330000000000000ull;
}
// a constant that stays in vector registers (and is not made anew for every use)
__device__ __forceinline__ double held_constant(double c) {
  asm volatile("" : "+v"(c));
  return c;
}

template <int D>
__device__ __forceinline__ double lane_xor_d(double v) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = static_cast<uint32_t>(lane_xor_dpp<D>(static_cast<int>(b)));
  const uint32_t hi = static_cast<uint32_t>(lane_xor_dpp<D>(static_cast<int>(b >> 32)));
  return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}
// The value of a lane with which this one shares a step of a sum over 2, 4, 8 or 16 lanes (where the steps before it have made equal what
// lies closer).  It is always there: no register is cleared for lanes that are not.
template <int STEP>
__device__ __forceinline__ int partner(int v) {
  constexpr int kCtrl = STEP == 1 ? 0xB1 : STEP == 2 ? 0x4E : STEP == 4 ? 0x141 : 0x128;  // lane ^ 1, ^ 2, 7 - lane of 8, 8 places on
  return __builtin_amdgcn_update_dpp(0, v, kCtrl, 0xf, 0xf, true);
}
template <int STEP>
__device__ __forceinline__ double partner(double v) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = static_cast<uint32_t>(partner<STEP>(static_cast<int>(b)));
  const uint32_t hi = static_cast<uint32_t>(partner<STEP>(static_cast<int>(b >> 32)));
  return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}
template <int LANES = 16>
__device__ __forceinline__ double row16_sum_d(double v) {
  v += partner<1>(v);
  v += partner<2>(v);
  v += partner<4>(v);
  if constexpr (LANES == 16) v += partner<8>(v);
  return v;
}
template <int LANES>
__device__ __forceinline__ int row16_max(int v) {
  v = max(v, partner<1>(v));
  v = max(v, partner<2>(v));
  v = max(v, partner<4>(v));
  return LANES == 16 ? max(v, partner<8>(v)) : v;
}
// floats as integers in the same order, and back (no NaN)
__device__ __forceinline__ int in_order(float v) {
  const int b = __builtin_bit_cast(int, v);
  return b ^ (b >> 31 & INT_MAX);
}
__device__ __forceinline__ float from_order(int b) { return __builtin_bit_cast(float, b ^ (b >> 31 & INT_MAX)); }
// The largest of N (the instruction itself: fmaxf would first quiet every operand); +infinity if one is a NaN
template <int N>
__device__ __forceinline__ float max_of(const float (&z)[N]) {
  float m = z[0];
  bool nan = false;
#pragma unroll
  for (int j = 0; j < N; j += 2) {
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(m) : "v"(m), "v"(z[j]), "v"(z[j + 1]));
    nan |= __builtin_isunordered(z[j], z[j + 1]);
  }
  return nan ? INFINITY : m;
}
__device__ __forceinline__ double wave_sum_d(double v) {
  v += lane_xor_d<32>(v);
  v += lane_xor_d<16>(v);
  return row16_sum_d(v);
}
// of a ballot, the bits of the lanes in front of this one
__device__ __forceinline__ int lanes_before(uint64_t hit) {
  return __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(hit >> 32), __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(hit), 0));
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
  // the lane's entries of several slots: the row's last one in place of those behind it
  template <int N>
  __device__ __forceinline__ void gather(const int (&slot)[N], int lane, float (&z)[N]) const {
#pragma unroll
    for (int k = 0; k < N; ++k) z[k] = logit(min(slot[k] * kSlot + lane, V - 1));
    if (penalties) {
#pragma unroll
      for (int k = 0; k < N; ++k) z[k] -= penalty(min(slot[k] * kSlot + lane, V - 1));
    }
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

// The buckets of the parts' histograms: places on one grid of kGrid to an octave, counted down from the largest entry's, so that those of
// different parts fit together; the last one holds whatever lies lower.  In 32 bits: a smaller z never has a higher place, and a difference
// of two places below kBuckets is exact (of whole numbers up to 2^24, or of two that lie within a factor of two); buckets need not be alike.
__device__ __forceinline__ float grid_place(float z, const Power& p) { return floorf(z * p.grid); }
// Octaves by which the powers of bucket b of a part are raised before they are rounded to units of 1 / kPartOne: beside a part's largest those far down,
// in the last bucket above all, keep their digits so.  Raised powers are at most 2: bucket b is b places below the largest entry's, so its
// entries are b - 1 or more below that entry, and less by what rounding makes of two places (2^-24 of either), which is less than seven as far
// as kFarthest.
__device__ __forceinline__ int part_raised(int b) { return static_cast<unsigned>(b) / kGrid; }
// From this place on rounding is not a matter of a few places: a part's sum is taken from its entries, and the row's cut looked for among them.  (That is
// where the temperature is some 10^-7 of the largest entry, and neighbouring numbers are octaves apart.)
constexpr float kFarthest = 33554432.0f;  // 2^25

// A block takes a part of a row in NT threads, each E neighbours at a time, which add up as sums of four, then those, then the slot's threads.
// Loads are as wide as they are apart, at any alignment.  What bounds it: the loads and what is computed, one after the other in a block and only in
// part beside one another (512 rows of 65536, us: loads and maxima alone 26, that is 5.1 TB/s; sums of the entries themselves 30; of their powers
// 40; histograms 45).  Four neighbours to a thread take more steps to a slot's sum: 256 rows of 65536 without filters 27.7 a call instead of 25.7,
// with top-p 56.5 instead of 54.7; 1024 threads for few parts gain nothing (1 to 16 rows 4.0 to 4.6 with either, 31 rows 6.6 instead of
// 5.1); several parts to a block, the next one requested ahead, took 10 % longer.
template <typename T>
__global__ __launch_bounds__(kStatsThreads) void draw_stats_kernel(DrawArgs a) {
  constexpr int NT = kStatsThreads, E = 8, NV = kPart / E / NT, kLanes = kSlot / E;
  typedef T vec_t __attribute__((ext_vector_type(4), aligned(sizeof(T))));  // (a load need not be aligned)
  typedef float pen_t __attribute__((ext_vector_type(4), aligned(sizeof(float))));
  __shared__ float most[NT / 64];
  __shared__ unsigned long long mass[kBuckets];
  __shared__ unsigned count[kBuckets];
  const int row = blockIdx.x, part = blockIdx.y;
  const Wish w = wish_of(a, row);
  if (!w.valid) return;
  const Row<T> r = row_of<T>(a, row, w.source);
  const bool sums = w.needs_sums(), histogram = w.needs_histogram(), counts = w.top_k != INT_MAX;
  const int first = part * kPart + threadIdx.x * E;
  float z[NV][E];
#pragma unroll
  for (int q = 0; q < NV; ++q) {
    const int i = first + q * NT * E;
    if (i + E <= a.V) {
#pragma unroll
      for (int k = 0; k < E; k += 4) {
        const vec_t l = *reinterpret_cast<const vec_t*>(r.logits + i + k);
#pragma unroll
        for (int j = 0; j < 4; ++j) z[q][k + j] = static_cast<float>(l[j]);
      }
      if (r.penalties) {
#pragma unroll
        for (int k = 0; k < E; k += 4) {
          const pen_t p = *reinterpret_cast<const pen_t*>(r.penalties + i + k);
#pragma unroll
          for (int j = 0; j < 4; ++j) z[q][k + j] -= p[j];
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < E; ++j) z[q][j] = r.logit(min(i + j, a.V - 1));
      if (r.penalties) {
#pragma unroll
        for (int j = 0; j < E; ++j) z[q][j] -= r.penalty(min(i + j, a.V - 1));
      }
#pragma unroll
      for (int j = 0; j < E; ++j) z[q][j] = i + j < a.V ? z[q][j] : -INFINITY;
    }
  }
  static_assert(NT >= kBuckets && NT % 64 == 0, "a thread for every bucket");
  if (histogram && threadIdx.x < kBuckets) {
    mass[threadIdx.x] = 0;
    count[threadIdx.x] = 0;
  }
  float m = -INFINITY;
#pragma unroll
  for (int q = 0; q < NV; ++q) {
    const int slot = (first + q * NT * E) / kSlot;
    const float mq = from_order(row16_max<kLanes>(in_order(max_of(z[q]))));  // (a NaN counts as +infinity: no distribution)
    if (threadIdx.x % kLanes == 0 && slot < a.slots) a.slot_max[static_cast<int64_t>(row) * a.slots + slot] = mq;
    m = fmaxf(m, mq);
  }
  if (!sums && !histogram) return;
  m = wave_reduce_dpp(m, [](float x, float y) { return fmaxf(x, y); });
  if ((threadIdx.x & 63) == 0) most[threadIdx.x >> 6] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < NT / 64; ++i) m = fmaxf(m, most[i]);
  m = scalar(m);
  const int64_t at = static_cast<int64_t>(row) * a.parts + part;
  if (threadIdx.x == 0) a.part_max[at] = m;
  const float top = scalar(grid_place(m, w.power));
  const double ninth = held_constant(kNinth), one = held_constant(kPartOne), two = held_constant(2.0 * kOne), round = held_constant(kRound);
  const auto slot_sum = [&](int q) {
    double sum = 0.0, four = 0.0;
#pragma unroll
    for (int j = 0; j < E; ++j) {
      four += weight(z[q][j], m, w.power, ninth, round);
      if (j % 4 == 3) {
        sum += four;
        four = 0.0;
      }
    }
    return row16_sum_d<kLanes>(sum);
  };
  if (sums) {
#pragma unroll
    for (int q = 0; q < NV; ++q) {
      const int slot = (first + q * NT * E) / kSlot;
      const double sum = slot_sum(q);
      if (threadIdx.x % kLanes == 0 && slot < a.slots) a.slot_sum[static_cast<int64_t>(row) * a.slots + slot] = sum;
    }
    return;
  }
#pragma unroll
  for (int q = 0; q < NV; ++q)
#pragma unroll
    for (int j = 0; j < E; ++j) {  // (-infinity, and whatever a row without a distribution holds: the last bucket, with nothing)
      const int b = static_cast<int>(fminf(top - grid_place(z[q][j], w.power), static_cast<float>(kBuckets - 1)));
      atomicAdd(&mass[b], in_units(weight<true>(z[q][j], m, w.power, ninth, round, part_raised(b)), one, two));
      if (counts) atomicAdd(&count[b], 1u);
    }
  // (sums of what the buckets hold: in one order, whatever order the entries came in)
  __syncthreads();
  const int b = threadIdx.x;
  const bool far = !(fabsf(top) < kFarthest);
  if (b < kBuckets) {
    const unsigned long long held = mass[b];
    a.part_mass[at * kBuckets + b] = held;
    if (counts) a.part_count[at * kBuckets + b] = count[b];
    const double sum = wave_sum_d(ldexp(static_cast<double>(held), -part_raised(b)));
    if ((b & 63) == 0 && !far) a.part_sum[at * kSums + b / 64] = sum;
  }
  if (!far) return;
  double* slots = reinterpret_cast<double*>(mass);
  __syncthreads();
#pragma unroll
  for (int q = 0; q < NV; ++q) {
    const double sum = slot_sum(q);
    if (threadIdx.x % kLanes == 0) slots[(threadIdx.x + q * NT) / kLanes] = sum;
  }
  __syncthreads();
  if (threadIdx.x >= 64) return;
  const double sum = wave_sum_d(slots[threadIdx.x]);
  if (threadIdx.x < kSums) a.part_sum[at * kSums + threadIdx.x] = threadIdx.x == 0 ? sum * kPartOne : 0.0;
}

// What one wavefront or thread finds for its block, and what wavefronts exchange: by the block functions, and at places of their own
template <int NW, int LIST>
struct Shared {
  static constexpr int kWaves = NW, kList = LIST;
  double d[NW], d2[NW], total[NW], chunk[NW];
  float f[NW], f2[NW], most[NW], least[NW];
  int i[NW], reach[NW], entries[NW];
  unsigned count[kBuckets];
  unsigned long long mass[kBuckets];
  unsigned carry[kBuckets];  // 2^64 of the mass
  float last_z[kLast];
  int last_i[kLast];
  alignas(8) float list_z[LIST];  // entries in order of their indexes
  int list_i[LIST];
  int bucket, bucket_count, at, slot;
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
  float octaves, first;  // of a bucket, and from m to the first one (a little less)
  __device__ __forceinline__ int of(float z) const {
    return static_cast<int>(fmin((top - static_cast<double>(z)) * per_unit, static_cast<double>(kBuckets - 1)));
  }
  // octaves by which all of a bucket lies below m, rounded down: by so many its powers are raised before they are rounded to units of 1 / kOne
  __device__ __forceinline__ int raised(int b) const { return static_cast<int>(fmaxf(fmaf(static_cast<float>(b), octaves, first), 0.0f)); }
};
// (`range` is at most 1000 octaves: an error of 32 bits in either term stays below the hundredth)
__device__ __forceinline__ Buckets buckets_of(double top, double range, float m, const Power& p) {
  range = fmax(range, 0.0);
  return {top, scalar(range > 0.0 ? kBuckets / range : 0.0), scalar(static_cast<float>(range * p.octaves / kBuckets)),
          scalar(static_cast<float>((static_cast<double>(m) - top) * p.octaves) - 0.01f)};
}

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
__device__ __forceinline__ void find_bucket(S& sh, const Cut& cut, const Buckets& buckets, int above, double above_mass, bool inside) {
  constexpr int kPer = kBuckets / 64;
  const int lane = threadIdx.x & 63;
  int n = 0;
  double masses[kPer], held = 0.0;
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const int b = lane * kPer + j;
    masses[j] = ldexp(fma(static_cast<double>(sh.carry[b]), 0x1p64, static_cast<double>(sh.mass[b])) * (1.0 / kOne), -buckets.raised(b));
    n += sh.count[b];
    held += masses[j];
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
    at_held += masses[j];
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
// the same.  Every bucket has a unit of its own, 2^-51 of the largest power that it can hold: of a row that is nearly sure the cut lies some forty
// octaves down, where a unit for all would leave few bits or none.  (The list's powers stay below 2^64 units, a row's are carried.)
template <typename S, typename R>
__device__ __forceinline__ bool find_cut(S& sh, const R* row, int c0, int c1, int n, const Cut& cut, float m, const Power& power, Span span,
                                         Buckets buckets, bool inside, Found& found) {
  constexpr int kThreads = S::kWaves * 64;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  static_assert(S::kList <= 8000, "the list's powers in units");
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
      sh.carry[b] = 0;
    }
    __syncthreads();
    each([&](float z) {
      const int b = buckets.of(z);
      atomicAdd(&sh.count[b], 1u);
      if (cut.mass < INFINITY) {
        const unsigned long long units = in_units(weight(z, m, power, kNinth, kRound, buckets.raised(b)));
        if (in_list) atomicAdd(&sh.mass[b], units);
        else if (atomicAdd(&sh.mass[b], units) > ~units) atomicAdd(&sh.carry[b], 1u);
      }
    });
    __syncthreads();
    if (wave == 0) find_bucket(sh, cut, buckets, span.above, span.above_mass, inside);
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
      const int want = equal ? equal_ones(cut, span.above, span.above_mass, count, weight(span.low, m, power)) : 0;
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
          if (__builtin_amdgcn_inverse_ballot_w64(hit)) take(z, i, place + lanes_before(hit));
          place += __popcll(hit);
        });
      }
      __syncthreads();
      if (last) {
        if (!equal && wave == 0) {
          const float z = lane < count ? sh.last_z[lane] : -INFINITY;
          const double e = weight(z, m, power);
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
    buckets = buckets_of(span.high, static_cast<double>(span.high) - static_cast<double>(span.low), m, power);
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
  const double e = weight(z, m, w.power);
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
  const double target = w.target(__shfl(upto, 63, 64));
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
      const double v = weight(z, m, w.power);
      if (found.keeps(z, sh.list_i[k]) && w.likely(v)) e[j] = v;
    }
    mine += e[j];
  }
  double kept;
  const double before = block_before(mine, sh.d, &kept);
  const double target = w.target(kept);
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
  if (tid == 0) answer(sh.list_i[at], static_cast<float>(-log1p(others / weight(sh.list_z[at], m, w.power))));
}

constexpr int kPickWaves = kPickThreads / 64;
constexpr int kMaxParts = kMaxLogprobVocab / kPart;
constexpr int kPartSlots = kPart / kSlot;
struct PickShared : Shared<kPickWaves, kList> {
  uint16_t slots[kPickWaves][kWaveSlots];
  double part_scale[kMaxParts];  // a part's largest power, by kPartOne
  int part_shift[kMaxParts];     // the part's first bucket, among the row's
  double held[kPickThreads];
  unsigned number[kPickThreads];
  double mass_at;
  int first, last;               // buckets of the window
};
static_assert(kMaxLogprobVocab / kSlot / kPickWaves * sizeof(double) <= kList * sizeof(float), "the sums of a chunk's slots lie where the list was");
static_assert(kPickThreads % kBuckets == 0, "so many threads for a bucket");

// The smallest float whose place on the grid is at least `place`; false: not found next to where it should be
__device__ __forceinline__ bool grid_edge(double place, const Power& p, float& z) {
  constexpr double kMax = FLT_MAX;
  z = p.grid > 0.0f ? static_cast<float>(fmin(fmax(place / p.grid, -kMax), kMax)) : -FLT_MAX;
  int left = 16;
  while (grid_place(z, p) >= place && z > -FLT_MAX && left > 0) {
    z = nextafterf(z, -INFINITY);
    --left;
  }
  while (grid_place(z, p) < place && z < FLT_MAX && left > 0) {
    z = nextafterf(z, INFINITY);
    --left;
  }
  return left > 0;
}

// The row's histogram out of its parts': the cut's sum, and the bucket in which the cut lies, or that of the least entry that min_p keeps
template <typename W>
__device__ __forceinline__ void place_window(const DrawArgs& a, PickShared& sh, int row, const W& w, float m, float top) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const float* part_max = a.part_max + static_cast<int64_t>(row) * a.parts;
  const double* part_sum = a.part_sum + static_cast<int64_t>(row) * a.parts * kSums;
  const unsigned long long* part_mass = a.part_mass + static_cast<int64_t>(row) * a.parts * kBuckets;
  const unsigned* part_count = a.part_count + static_cast<int64_t>(row) * a.parts * kBuckets;
  const bool counts = w.top_k != INT_MAX;
  double mine = 0.0;
  for (int p = tid; p < a.parts; p += kPickThreads) {
    const float mp = part_max[p];
    const double scale = weight(mp, m, w.power);
    double sum = 0.0;
#pragma unroll
    for (int k = 0; k < kSums; ++k) sum += part_sum[p * kSums + k];
    sh.part_scale[p] = scale / kPartOne;
    mine += sum * sh.part_scale[p];
    sh.part_shift[p] = mp > -INFINITY ? static_cast<int>(fminf(top - grid_place(mp, w.power), static_cast<float>(kBuckets))) : kBuckets;
  }
  mine = wave_sum_d(mine);
  if (lane == 0) sh.total[wave] = mine;
  __syncthreads();
  // bucket b of a part is the row's bucket b + shift; a part's last one says nothing but "lower"
  constexpr int kGroups = kPickThreads / kBuckets;
  const int j = tid % kBuckets;
  double held = 0.0;
  unsigned number = 0;
  if (j < kBuckets - 1) {
#pragma unroll 8
    for (int p = tid / kBuckets; p < a.parts; p += kGroups) {
      const int b = j - sh.part_shift[p];
      if (b >= 0) {
        held += ldexp(static_cast<double>(part_mass[p * kBuckets + b]) * sh.part_scale[p], -part_raised(b));
        if (counts) number += part_count[p * kBuckets + b];
      }
    }
  }
  sh.held[tid] = held;
  sh.number[tid] = number;
  __syncthreads();
  if (wave == 0) {
    constexpr int kPer = kBuckets / 64;
    double total = 0.0;
#pragma unroll
    for (int i = 0; i < kPickWaves; ++i) total += sh.total[i];
    const Cut cut = {w.top_k, w.top_p < 1.0 ? w.top_p * total : INFINITY};
    int numbers[kPer], all = 0;
    double sums[kPer], all_held = 0.0;
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      numbers[k] = 0;
      sums[k] = 0.0;
#pragma unroll
      for (int g = 0; g < kGroups; ++g) {
        numbers[k] += sh.number[g * kBuckets + lane * kPer + k];
        sums[k] += sh.held[g * kBuckets + lane * kPer + k];
      }
      all += numbers[k];
      all_held += sums[k];
    }
    int at = wave_upto(all) - all;
    const double upto = wave_upto(all_held);
    double at_held = __shfl_up(upto, 1, 64);
    if (lane == 0) at_held = 0.0;
    int cut_at = kBuckets;
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      sh.count[lane * kPer + k] = at;  // (in front of the bucket)
      sh.held[lane * kPer + k] = at_held;
      at += numbers[k];
      at_held += sums[k];
      if (cut_at == kBuckets && cut.reached(at, at_held)) cut_at = lane * kPer + k;
    }
    cut_at = wave_reduce_dpp(cut_at, [](int x, int y) { return min(x, y); });
    // and the buckets of an entry that min_p surely keeps and of one that it surely does not
    int kept_at = kBuckets, dropped_at = kBuckets;
    if (w.min_p > 0.0) {
      const double edge = log2(w.min_p);
      const auto bucket = [&](float z) { return static_cast<int>(fminf(fmaxf(top - grid_place(z, w.power), 0.0f), static_cast<float>(kBuckets))); };
      kept_at = bucket(nextafterf(static_cast<float>(m + (edge + 1e-3) / w.power.octaves), INFINITY));
      dropped_at = bucket(nextafterf(static_cast<float>(m + (edge - 1e-3) / w.power.octaves), -INFINITY));
    }
    if (lane == 0) {
      sh.mass_at = cut.mass;
      sh.first = min(cut_at, kept_at);
      sh.last = min(cut_at, dropped_at);
    }
  }
  __syncthreads();
}

// The entries from `low` up to `high`, from the slots that reach it, to the list, in order; what lies above them is known from the
// histograms, for every wavefront's chunk of the row.  False: the list is too short.  sh.reach: where each wavefront's begin
template <typename T>
__device__ __forceinline__ bool list_window(const DrawArgs& a, PickShared& sh, const Row<T>& r, int row, int c0, int c1, int first, float low, float high,
                                            int& n, double& kept_above) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const unsigned long long* part_mass = a.part_mass + static_cast<int64_t>(row) * a.parts * kBuckets;
  kept_above = 0.0;
  if (first > 0) {
#pragma unroll 2
    for (int s = c0; s < c1; s += kPartSlots) {
      const int p = s / kPartSlots, end = first - sh.part_shift[p];
      unsigned long long held[kSums];
#pragma unroll
      for (int k = 0; k < kSums; ++k) held[k] = part_mass[p * kBuckets + k * 64 + lane];
      double sum = 0.0;
#pragma unroll
      for (int k = 0; k < kSums; ++k) {
        const int b = k * 64 + lane;
        sum += b < end ? ldexp(static_cast<double>(held[k]), -part_raised(b)) : 0.0;
      }
      kept_above += sum * sh.part_scale[p];
    }
    kept_above = wave_sum_d(kept_above);
  }
  // each wavefront's to a share of the list
  constexpr int kShare = kList / kPickWaves;
  const float* slot_max = a.slot_max + static_cast<int64_t>(row) * a.slots;
  float* share_z = sh.list_z + wave * kShare;
  int* share_i = sh.list_i + wave * kShare;
  int inside = 0;
  constexpr int kAhead = 16;  // slots at once
  for (int s = c0; s < c1; s += 64) {
    const uint64_t reach = __ballot(s + lane < c1 && slot_max[min(s + lane, c1 - 1)] >= low);
#pragma unroll 1
    for (int g = 0; g < 64; g += kAhead) {
      if ((reach >> g & ((1ull << kAhead) - 1)) == 0) continue;
      const int i0 = (s + g) * kSlot + lane;
      float z[kAhead];
      r.template load<kAhead>(i0, z, 0);
      const int end = min(c1 * kSlot, a.V);
      if ((s + g + kAhead) * kSlot > end) {
#pragma unroll
        for (int k = 0; k < kAhead; ++k) z[k] = i0 + k * kSlot < end ? z[k] : -INFINITY;
      }
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        // (those too many fall on the last place: then the share is too short anyhow)
        const uint64_t hit = __ballot(z[k] >= low) & __ballot(z[k] < high);
        const int to = min(inside + lanes_before(hit), kShare - 1);
        if (__builtin_amdgcn_inverse_ballot_w64(hit)) {
          share_z[to] = z[k];
          share_i[to] = i0 + k * kSlot;
        }
        inside += __popcll(hit);
      }
    }
  }
  if (lane == 0) sh.entries[wave] = inside;
  __syncthreads();
  int all = 0, place = 0, widest = 0;
#pragma unroll
  for (int i = 0; i < kPickWaves; ++i) {
    if (i == wave) place = all;
    all += sh.entries[i];
    widest = max(widest, sh.entries[i]);
  }
  if (widest > kShare) return false;
  // the shares move together
  float z[kShare / 64];
  int i[kShare / 64];
#pragma unroll
  for (int k = 0; k < kShare / 64; ++k) {
    z[k] = sh.list_z[wave * kShare + k * 64 + lane];
    i[k] = sh.list_i[wave * kShare + k * 64 + lane];
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kShare / 64; ++k)
    if (k * 64 + lane < inside) {
      sh.list_z[place + k * 64 + lane] = z[k];
      sh.list_i[place + k * 64 + lane] = i[k];
    }
  sh.reach[wave] = place;
  n = scalar(all);
  __syncthreads();
  return true;
}

// A block draws for a row.  What bounds it is the chain of its steps, each a trip to memory or a few hundred instructions between barriers: V =
// 65536 with top_k 20 and top_p 10 us (maxima 1.6, bound 2.8, slots 0.8, list 2), with top-p over a flat row 28 (window 4, listing 10, cut 4, sums
// 10).  512 threads whatever the batch is, so that sums split alike; two blocks to a CU: 512 rows at once, whose chains fill one another's
// waits (45 us).
template <typename T>
__global__ __launch_bounds__(kPickThreads, 4) void draw_pick_kernel(DrawArgs a) {  // (four wavefronts per SIMD: two blocks per CU)
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

  const float* part_max = a.part_max + static_cast<int64_t>(row) * a.parts;
  // (0 for a slot whose entries all lie below every power, though its part's largest does not: none of them could be drawn)
  const auto slot_share = [&](int s) {
    const double share = slot_sum[s] * weight(part_max[s / (kPart / kSlot)], m, w.power);
    return static_cast<double>(slot_max[s]) - m >= w.power.lowest ? share : 0.0;
  };
  double mine = 0.0;

  if (w.free()) {
    // by the slots' sums the slot, then its entry
    for (int s = s0; s < s1; ++s) mine += slot_share(s);
    double kept;
    const double before = block_before(mine, sh.d, &kept);
    const double target = w.target(kept);
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
    if (wave == 0) draw_entry([&](float z, int) { return weight(z, m, w.power); }, r, slot, sh.before, target, others, answer);
    return;
  }

  // How far down a kept entry can lie.  Rows with histograms: to the end of the window in which the last one is; others: as far as the
  // slots say.
  const bool histogram = w.needs_histogram();
  Cut cut = {w.top_k, INFINITY};
  float low = -FLT_MAX, high = INFINITY;
  int first = 0;
  bool told = false;  // the window is known
  if (histogram) {
    const float top = grid_place(m, w.power);
    place_window(a, sh, row, w, m, top);
    cut.mass = scalar(sh.mass_at);
    first = scalar(sh.first);
    const int last = scalar(sh.last);
    const double from = top;
    told = fabsf(top) < kFarthest && last < kBuckets - 1 && grid_edge(from - last, w.power, low) && (first == 0 || grid_edge(from - first + 1.0, w.power, high));
    if (!told) low = -FLT_MAX;
  } else {
    const bool summed = w.needs_sums();
    double range = scalar(static_cast<double>(m) - static_cast<double>(lowest));
    if (range * w.power.octaves > kWidest) range = kWidest / w.power.octaves;
    const Buckets rough = buckets_of(m, scalar(range), m, w.power);
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
    cut.mass = scalar(w.top_p < 1.0 ? w.top_p * total : INFINITY);
    const double width = scalar(range * w.power.octaves / kBuckets);  // octaves of a bucket
    const auto edge = [&](int b) { return __builtin_amdgcn_exp2f(static_cast<float>(-(b + 1) * width)); };  // the least power of a bucket
    if (wave == 0) {
      // Bucket b bounds the kept entries if, of the entries up to it, there are top_k (as many slots reach it), or top_p (what is in other
      // slots, and what their own entries below the bucket can hold at most, or all entries of the row, is less than the rest), or all that
      // min_p keeps.
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
      int bound = kBuckets - 1;
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        const int b = lane * kPer + j;
        at += sh.count[b];
        at_held += static_cast<double>(sh.mass[b]) * kUnit;
        bool enough = at >= w.top_k || (b + 1) * width > unlikely;
        if (summed) enough |= fmin(total - at_held + static_cast<double>(at) * kSlot * edge(b) * 1.001, a.V * 1.001 * edge(b)) <= spare;
        if (enough) bound = min(bound, b);
      }
      bound = wave_reduce_dpp(bound, [](int x, int y) { return min(x, y); });
      if (lane == 0) sh.bucket = bound;
    }
    __syncthreads();
    const int bound = scalar(sh.bucket);
    if (bound < kBuckets - 1) low = fmaxf(nextafterf(static_cast<float>(m - (bound + 1) * range / kBuckets), -INFINITY), -FLT_MAX);
  }
  // Entries below every power change neither the token nor a sum (masks of a finite value: 64 rows of 65536 with 30 entries that are not
  // masked, top_k 50: 15 us instead of 143).
  low = fmaxf(low, nextafterf(static_cast<float>(m + w.power.lowest), -INFINITY));
  const auto candidate = [&](float z) { return z >= low; };

  // the slots that reach the bound, each wavefront its own
  int reach = 0, n = 0;
  for (int s = s0; s < s1; ++s) reach += candidate(slot_max[s]);
  const int reach_upto = wave_upto(reach);
  const int mine_reach = __builtin_amdgcn_readlane(reach_upto, 63);
  if (lane == 0) sh.reach[wave] = mine_reach;
  __syncthreads();
  int all = 0, widest = 0;
#pragma unroll
  for (int i = 0; i < kPickWaves; ++i) {
    all += sh.reach[i];
    widest = max(widest, sh.reach[i]);
  }
  all = scalar(all);
  widest = scalar(widest);
  bool fits = widest <= kWaveSlots && (!told || all <= kMost);
  if (fits) {
    // in order; their entries kHeld slots at a time, the first of which stay in registers
    uint16_t* own = sh.slots[wave];
    for (int s = s0, to = reach_upto - reach; s < s1; ++s)
      if (candidate(slot_max[s])) own[to++] = static_cast<uint16_t>(s);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    const auto load = [&](int k0, int (&slot)[kHeld], float (&z)[kHeld]) {
#pragma unroll
      for (int k = 0; k < kHeld; ++k) slot[k] = own[min(k0 + k, mine_reach - 1)];
      r.gather(slot, lane, z);
#pragma unroll
      for (int k = 0; k < kHeld; ++k) z[k] = k0 + k < mine_reach && slot[k] * kSlot + lane < a.V ? z[k] : -INFINITY;
    };
    int slot[kHeld], place = 0, entries = 0;
    float held[kHeld];
    if (mine_reach > 0) load(0, slot, held);
    for (int k0 = 0; k0 < mine_reach;) {
      if (k0 > 0) load(k0, slot, held);
#pragma unroll
      for (int k = 0; k < kHeld; ++k) entries += __popcll(__ballot(candidate(held[k])));
      k0 += kHeld;
    }
    if (lane == 0) sh.i[wave] = entries;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kPickWaves; ++i) {
      if (i == wave) place = n;
      n += sh.i[i];
    }
    n = scalar(n);
    fits = n <= kList;
    if (fits) {
      for (int k0 = 0; k0 < mine_reach; k0 += kHeld) {
        if (mine_reach > kHeld) load(k0, slot, held);
#pragma unroll
        for (int k = 0; k < kHeld; ++k) {
          const uint64_t hit = __ballot(candidate(held[k]));
          if (__builtin_amdgcn_inverse_ballot_w64(hit)) {
            const int to = place + lanes_before(hit);
            sh.list_z[to] = held[k];
            sh.list_i[to] = slot[k] * kSlot + lane;
          }
          place += __popcll(hit);
        }
      }
    }
  }
  if (fits) {
    __syncthreads();
    if (n <= 64) {
      if (wave == 0) draw_from_few(sh, n, w, cut, m, answer);
      return;
    }
    Found found = {-INFINITY, INT_MAX};
    if (!cut.open())
      find_cut(sh, static_cast<const Row<T>*>(nullptr), 0, 0, n, cut, m, w.power, {0, 0.0, -FLT_MAX, FLT_MAX},
               buckets_of(m, fmin(static_cast<double>(m) - low, kWidest / w.power.octaves), m, w.power), false, found);
    draw_from_list(sh, n, w, found, m, answer);
    return;
  }

  // Many candidates.  The cut is looked for in the window alone; where that is wider than the list, or not known, in memory.
  const int chunk = (a.parts + kPickWaves - 1) / kPickWaves * kPartSlots;  // slots of a wavefront: whole parts
  const int c0 = min(wave * chunk, a.slots), c1 = min(c0 + chunk, a.slots);
  Found found = {-INFINITY, INT_MAX};
  Span span = {0, 0.0, low, FLT_MAX};
  double kept_above = 0.0;
  bool windowed = false;
  if (told) {
    if (high < INFINITY) span.high = nextafterf(high, -INFINITY);
    span.above = scalar(static_cast<int>(sh.count[first]));
    span.above_mass = scalar(sh.held[first]);
    windowed = list_window(a, sh, r, row, c0, c1, first, low, high, n, kept_above);
  }
  if (!cut.open()) {
    const double from = fmin(span.high, m);
    find_cut(sh, windowed ? nullptr : &r, c0, c1, windowed ? n : 0, cut, m, w.power, span,
             buckets_of(from, fmin(from - span.low, kWidest / w.power.octaves), m, w.power), false, found);
  }

  // the kept entries' sums by wavefronts, of the entry's wavefront by slots, of its slot by entries
  // (nothing below the window, in which the histograms say the last one is: where sums that are rounded otherwise do not reach the cut there,
  // it is the window's last entry)
  const auto kept_weight = [&](float z, int i) {
    const double e = weight(z, m, w.power);
    return z >= span.low && found.keeps(z, i) && w.likely(e) ? e : 0.0;
  };
  double share = 0.0;
  if (windowed) {
    // (a list in order: this wavefront's part of it is what lies in its chunk)
    share = lane == 0 ? kept_above : 0.0;
    const int end = wave + 1 < kPickWaves ? sh.reach[wave + 1] : n;
    for (int k = sh.reach[wave] + lane; k < end; k += 64) share += kept_weight(sh.list_z[k], sh.list_i[k]);
  } else {
    share = lane == 0 ? kept_above : 0.0;
    each_entry(r, c0, c1, [&](float z, int i) {
      if (z >= span.low && z <= span.high) share += kept_weight(z, i);
    });
  }
  share = wave_sum_d(share);
  __syncthreads();
  if (lane == 0) sh.chunk[wave] = share;
  __syncthreads();
  double kept = 0.0;
#pragma unroll
  for (int i = 0; i < kPickWaves; ++i) kept += sh.chunk[i];
  const double target = w.target(kept);
  double upto = 0.0, before = 0.0, others = 0.0;
  int owner = -1;
  bool sure = false;
#pragma unroll
  for (int i = 0; i < kPickWaves; ++i) {
    const double v = sh.chunk[i];
    if (v > 0.0 && !sure) {
      owner = i;
      before = upto;
      sure = upto + v > target;
    }
    upto += v;
  }
#pragma unroll
  for (int i = 0; i < kPickWaves; ++i) others += i == owner ? 0.0 : sh.chunk[i];
  const int o0 = owner * chunk, slots = min(o0 + chunk, a.slots) - o0;
  double* sums = reinterpret_cast<double*>(sh.list_z);
  // (16 lanes a slot: four entries each, then four steps to their sum)
  for (int s = wave * 4; s < slots; s += 4 * kPickWaves) {
    const int own = o0 + min(s + lane / 16, slots - 1);
    double sum = 0.0;
    float z[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) z[k] = r.at(own * kSlot + k * 16 + lane % 16);
#pragma unroll
    for (int k = 0; k < 4; ++k) sum += kept_weight(z[k], own * kSlot + k * 16 + lane % 16);
    sum = row16_sum_d(sum);
    if (lane % 16 == 0) sums[own - o0] = sum;
  }
  __syncthreads();
  if (wave != 0) return;
  // one wavefront over a chunk's sums (up to kMaxLogprobVocab / kSlot / kPickWaves), 64 at a time
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
// Bound by memory (64 rows of 65536: 6 us, 5.6 TB/s); all of a thread's entries are requested ahead of its first store.  (Entries behind the row's
// end are read as its last one, which another thread may have written already where out is penalties: what they hold is not used.)
constexpr int kEach = 8;  // entries of a thread
__global__ __launch_bounds__(256) void draw_penalties_kernel(int V, const float* penalties, float* out, const int* token, const float* presence,
                                                             const float* frequency, const float* decay) {
  const int row = blockIdx.x;
  const int pick = token[row];
  const float keep = decay ? decay[row] : 1.0f;
  const float once = presence ? presence[row] : 0.0f, again = frequency ? frequency[row] : 0.0f;
  const int64_t base = static_cast<int64_t>(row) * V;
  const int first = blockIdx.y * kEach * 256 + threadIdx.x;
  float p[kEach];
#pragma unroll
  for (int k = 0; k < kEach; ++k) p[k] = penalties[base + min(first + k * 256, V - 1)];
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    const int i = first + k * 256;
    if (i < V) out[base + i] = fmaf(p[k], keep, i != pick ? 0.0f : p[k] == 0.0f ? once : again);
  }
}

template <typename T>
void launch_draw(hipStream_t st, int rows, const DrawArgs& a) {
  hipLaunchKernelGGL((draw_stats_kernel<T>), dim3(rows, a.parts), dim3(kStatsThreads), 0, st, a);
  hipLaunchKernelGGL((draw_pick_kernel<T>), dim3(rows), dim3(kPickThreads), 0, st, a);
}

// The arrays of a workspace, one after the other, those of 8 bytes first
DrawArgs lay_out(DrawArgs a, int rows, void* workspace, size_t* bytes) {
  a.slots = ceil_div(a.V, kSlot);
  a.parts = ceil_div(a.V, kPart);
  char* at = static_cast<char*>(workspace);
  const auto take = [&](auto*& p, size_t n) {
    p = reinterpret_cast<std::remove_reference_t<decltype(p)>>(at);
    at += n * sizeof(*p);
  };
  const size_t slots = static_cast<size_t>(rows) * a.slots, parts = static_cast<size_t>(rows) * a.parts;
  take(a.slot_sum, slots);
  take(a.part_sum, parts * kSums);
  take(a.part_mass, parts * kBuckets);
  take(a.slot_max, slots);
  take(a.part_max, parts);
  take(a.part_count, parts * kBuckets);
  *bytes = (static_cast<size_t>(at - static_cast<char*>(workspace)) + 15) / 16 * 16;
  return a;
}

}  // namespace

}  // namespace rwkv

using namespace rwkv;

extern "C" {

int rwkv_hip_draw_tokens_workspace(int rows, int V, size_t* bytes) {
  RWKV_REQUIRE(bytes && rows > 0 && V > 0 && V <= kMaxLogprobVocab, "draw_tokens_workspace: bad arguments");
  DrawArgs a = {};
  a.V = V;
  lay_out(a, rows, nullptr, bytes);
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
  DrawArgs a = {};
  a.logits = logits;
  a.ld = ld;
  a.V = V;
  a.logit_rows = logit_rows;
  a.source = static_cast<const int*>(source);
  a.temperature = static_cast<const float*>(temperature);
  a.top_k = static_cast<const int*>(top_k);
  a.top_p = static_cast<const float*>(top_p);
  a.min_p = static_cast<const float*>(min_p);
  a.uniform = static_cast<const float*>(uniform);
  a.penalties = static_cast<const float*>(penalties);
  a.token = static_cast<int*>(token);
  a.logprob = static_cast<float*>(logprob);
  size_t need = 0;
  a = lay_out(a, rows, workspace, &need);
  RWKV_REQUIRE(workspace && workspace_bytes >= need && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0,
               "draw_tokens: workspace of %zu bytes (aligned to 16) needed, got %zu", need, workspace_bytes);
  if (io == RWKV_IO_F16) launch_draw<half_t>(as_stream(s), rows, a);
  else launch_draw<float>(as_stream(s), rows, a);
  if (penalties_out)
    hipLaunchKernelGGL(draw_penalties_kernel, dim3(rows, ceil_div(V, kEach * 256)), dim3(256), 0, as_stream(s), V, static_cast<const float*>(penalties),
                       static_cast<float*>(penalties_out), static_cast<const int*>(token), static_cast<const float*>(presence),
                       static_cast<const float*>(frequency), static_cast<const float*>(decay));
  RWKV_LAUNCH_CHECK();
  return RWKV_OK;
}

}  // extern "C"
