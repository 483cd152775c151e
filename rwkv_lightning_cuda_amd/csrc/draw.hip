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
// Two launches.  draw_stats_kernel reads the rows with the whole chip: per 64 entries (a slot) the largest z and, where the
// sum over the whole row is asked for, the sum of the slot's powers.  draw_pick_kernel has a block per row: the slots bound how small a kept
// entry can be, the slots that reach the bound are read again, and the entries above it go to a list in LDS, in order.  Lists are
// short for the filters that servers use.  A row whose list overflows (flat rows with top-p alone, a large top-k, many equal logits) is searched in
// memory instead, and one without filters needs no list: its slots' sums give the token's slot.
#include <cfloat>
#include <climits>
#include <type_traits>

#include "ops.h"

namespace rwkv {

namespace {

constexpr int kSlot = 64;
constexpr int kStatsThreads = 256;
constexpr int kPickThreads = 1024;
constexpr int kPickWaves = kPickThreads / 64;
constexpr int kBuckets = 256;   // of a histogram
constexpr int kList = 4096;     // entries
constexpr int kLast = 64;       // entries that one wavefront puts in order
constexpr double kLog2eD = 1.44269504088896340736;
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
  double* slot_sum;  // [rows,slots]
  float* slot_max;   // [rows,slots]
};

// What a row asks for.  Filters that are off: top_k = INT_MAX, top_p >= 1, min_p <= 0.
struct Wish {
  double octaves;  // log2(e) / temperature
  double top_p, min_p, u;
  int top_k, source;
  bool valid, greedy;
  __device__ __forceinline__ bool free() const { return top_k == INT_MAX && top_p >= 1.0 && min_p <= 0.0; }
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
  w.octaves = w.greedy ? 0.0 : kLog2eD / static_cast<double>(t);
  return w;
}

// 2^y for y <= 0: the power series of e^(f ln 2) for |f| <= 1/2 up to the 12th power (the next term is 2e-16 there)
__device__ __forceinline__ double power(double y) {
  const double n = rint(y);
  const double f = (y - n) * 0.693147180559945309417;
  double p = 1.0 / 479001600.0;
  p = fma(p, f, 1.0 / 39916800.0);
  p = fma(p, f, 1.0 / 3628800.0);
  p = fma(p, f, 1.0 / 362880.0);
  p = fma(p, f, 1.0 / 40320.0);
  p = fma(p, f, 1.0 / 5040.0);
  p = fma(p, f, 1.0 / 720.0);
  p = fma(p, f, 1.0 / 120.0);
  p = fma(p, f, 1.0 / 24.0);
  p = fma(p, f, 1.0 / 6.0);
  p = fma(p, f, 0.5);
  p = fma(p, f, 1.0);
  p = fma(p, f, 1.0);
  return y < kLowestPower ? 0.0 : ldexp(p, static_cast<int>(n));
}
// e of an entry z <= m
__device__ __forceinline__ double weight(float z, float m, double octaves) {
  if (!(z > -INFINITY)) return 0.0;
  return power((static_cast<double>(z) - static_cast<double>(m)) * octaves);
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

// entry i of a row, or -infinity behind its end
template <typename T>
struct Row {
  const T* logits;
  const float* penalties;
  int V;
  __device__ __forceinline__ float at(int i) const {
    if (i >= V) return -INFINITY;
    const float z = static_cast<float>(logits[i]);
    return penalties ? z - penalties[i] : z;
  }
};
template <typename T>
__device__ __forceinline__ Row<T> row_of(const DrawArgs& a, int row, int source) {
  return {static_cast<const T*>(a.logits) + source * a.ld, a.penalties ? a.penalties + static_cast<int64_t>(row) * a.V : nullptr, a.V};
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
      if (m > -INFINITY && m < INFINITY) {
#pragma unroll
        for (int j = 0; j < 4; ++j) sum += weight(z[q][j], m, w.octaves);
      }
      sum = row16_sum_d(sum);
    }
    if ((threadIdx.x & 15) == 0 && slot < a.slots) {
      const int64_t at = static_cast<int64_t>(row) * a.slots + slot;
      a.slot_max[at] = m;
      if (sums) a.slot_sum[at] = sum;
    }
  }
}

struct PickShared {
  double d[kPickWaves];
  double d2[kPickWaves];
  float f[kPickWaves];
  float f2[kPickWaves];
  int i[kPickWaves];
  unsigned count[kBuckets];
  unsigned long long mass[kBuckets];
  float last_z[kLast];
  int last_i[kLast];
  float list_z[kList];
  int list_i[kList];
  uint16_t slots[kList];
  // what one wavefront or thread finds for the block
  int bucket, bucket_count, at, slot;
  double above_mass, before;
  float cut_z;
  int cut_i;
};

template <typename Op>
__device__ __forceinline__ float block_all(float v, Op op, float* buf) {
  v = wave_reduce_dpp(v, op);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) buf[threadIdx.x >> 6] = v;
  __syncthreads();
  float r = buf[0];
#pragma unroll
  for (int i = 1; i < kPickWaves; ++i) r = op(r, buf[i]);
  return r;
}
__device__ __forceinline__ int block_min(int v, int* buf) {
  v = wave_reduce_dpp(v, [](int x, int y) { return min(x, y); });
  __syncthreads();
  if ((threadIdx.x & 63) == 0) buf[threadIdx.x >> 6] = v;
  __syncthreads();
  int r = buf[0];
#pragma unroll
  for (int i = 1; i < kPickWaves; ++i) r = min(r, buf[i]);
  return r;
}
__device__ __forceinline__ double block_sum_d(double v, double* buf) {
  v = wave_sum_d(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) buf[threadIdx.x >> 6] = v;
  __syncthreads();
  double r = 0.0;
#pragma unroll
  for (int i = 0; i < kPickWaves; ++i) r += buf[i];
  return r;
}
// sum over the threads in front of this one, and over all
template <typename T>
__device__ __forceinline__ T block_before(T v, T* buf, T* total) {
  const T upto = wave_upto(v);
  T before = __shfl_up(upto, 1, 64);
  if ((threadIdx.x & 63) == 0) before = T(0);
  __syncthreads();
  if ((threadIdx.x & 63) == 63) buf[threadIdx.x >> 6] = upto;
  __syncthreads();
  T base = T(0), all = T(0);
#pragma unroll
  for (int i = 0; i < kPickWaves; ++i) {
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
__device__ __forceinline__ Buckets buckets_of(double top, double range) { return {top, range > 0.0 ? kBuckets / range : 0.0}; }

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

// One wavefront over a histogram: the first bucket in which the cut lies, the entries and the mass in front of it.  Where the sums do not
// reach the cut: kBuckets, or the last bucket that holds anything (`inside`: the cut is known to lie in this histogram, and rounding hides it).
__device__ __forceinline__ void find_bucket(PickShared& sh, const Cut& cut, int above, double above_mass, double unit, bool inside) {
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
  const float* slot_max = a.slot_max + static_cast<int64_t>(row) * a.slots;
  double* slot_sum = a.slot_sum + static_cast<int64_t>(row) * a.slots;
  // a thread has neighbouring slots
  const int per = (a.slots + kPickThreads - 1) / kPickThreads;
  const int s0 = min(tid * per, a.slots), s1 = min(s0 + per, a.slots);
  float m = -INFINITY;
  if (w.valid)
    for (int s = s0; s < s1; ++s) m = fmaxf(m, slot_max[s]);
  m = block_all(m, fmax_op, sh.f);
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

  double mine = 0.0, total = 0.0;
  if (w.needs_sum()) {
    for (int s = s0; s < s1; ++s) mine += slot_sum[s] * weight(slot_max[s], m, w.octaves);
    total = block_sum_d(mine, sh.d);
  }
  const Cut cut = {w.top_k, w.top_p < 1.0 ? w.top_p * total : INFINITY};
  const auto likely = [&](double e) { return !(w.min_p > 0.0) || e >= w.min_p; };
  Found found = {-INFINITY, INT_MAX};
  bool listed = false;  // the candidates are in the list
  int n = 0;            // entries of the list

  if (!w.free()) {
    // how far down a kept entry can lie, from the slots
    float lowest = INFINITY;
    for (int s = s0; s < s1; ++s)
      if (slot_max[s] > -INFINITY) lowest = fminf(lowest, slot_max[s]);
    if (tid < kBuckets) {
      sh.count[tid] = 0;
      sh.mass[tid] = 0;
    }
    lowest = block_all(lowest, fmin_op, sh.f2);
    double range = static_cast<double>(m) - static_cast<double>(lowest);
    if (range * w.octaves > kWidest) range = kWidest / w.octaves;
    const Buckets rough = buckets_of(m, range);
    constexpr double kUnit = 1.0 / (1ll << 40);  // (a row's sum is at most 2^20)
    for (int s = s0; s < s1; ++s) {
      if (!(slot_max[s] > -INFINITY)) continue;
      const int b = rough.of(slot_max[s]);
      atomicAdd(&sh.count[b], 1u);
      if (cut.mass < INFINITY) atomicAdd(&sh.mass[b], static_cast<unsigned long long>(slot_sum[s] * weight(slot_max[s], m, w.octaves) * (1.0 / kUnit)));
    }
    __syncthreads();
    if (wave == 0) {
      // Bucket b bounds the kept entries if, of the entries up to it, there are top_k (as many slots reach it), or top_p (what is in other
      // slots, and what their own entries below the bucket can hold at most, is less than the rest), or all that min_p keeps.
      constexpr int kPer = kBuckets / 64;
      const double width = range * w.octaves / kBuckets;  // octaves of a bucket
      const double spare = (1.0 - w.top_p) * total - 1e-8 * total;
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
        bool enough = at >= w.top_k;
        if (cut.mass < INFINITY) enough |= total - at_held + static_cast<double>(at) * kSlot * power(-(b + 1) * width) <= spare;
        if (w.min_p > 0.0) enough |= (b + 1) * width > 1e-9 - log2(w.min_p);
        if (enough) bound = min(bound, b);
      }
      bound = wave_reduce_dpp(bound, [](int x, int y) { return min(x, y); });
      if (lane == 0) sh.bucket = bound;
    }
    __syncthreads();
    const int bound = sh.bucket;
    const auto candidate = [&](float z) { return z > -INFINITY && rough.of(z) <= bound; };

    // the slots that reach it, in order
    int reach = 0;
    for (int s = s0; s < s1; ++s) reach += candidate(slot_max[s]);
    int all;
    int at = block_before(reach, sh.i, &all);
    if (all <= kList) {
      for (int s = s0; s < s1; ++s)
        if (candidate(slot_max[s])) sh.slots[at++] = static_cast<uint16_t>(s);
      __syncthreads();
      // and their entries: each wavefront a run of slots, counted, then written
      const int run = (all + kPickWaves - 1) / kPickWaves;
      const int g0 = min(wave * run, all), g1 = min(g0 + run, all);
      constexpr int kHeld = 8;  // slots that stay in registers between the two
      float held[kHeld];
#pragma unroll
      for (int k = 0; k < kHeld; ++k) held[k] = g0 + k < g1 ? r.at(sh.slots[g0 + k] * kSlot + lane) : -INFINITY;
      int entries = 0;
#pragma unroll
      for (int k = 0; k < kHeld; ++k) entries += __popcll(__ballot(candidate(held[k])));
      for (int g = g0 + kHeld; g < g1; ++g) entries += __popcll(__ballot(candidate(r.at(sh.slots[g] * kSlot + lane))));
      __syncthreads();
      if (lane == 0) sh.i[wave] = entries;
      __syncthreads();
      int place = 0;
#pragma unroll
      for (int i = 0; i < kPickWaves; ++i) {
        if (i == wave) place = n;
        n += sh.i[i];
      }
      if (n <= kList) {
        listed = true;
        const auto put = [&](float z, int slot) {
          const bool is = candidate(z);
          const uint64_t hit = __ballot(is);
          if (is) {
            const int to = place + __popcll(hit & ((1ull << lane) - 1));
            sh.list_z[to] = z;
            sh.list_i[to] = slot * kSlot + lane;
          }
          place += __popcll(hit);
        };
#pragma unroll
        for (int k = 0; k < kHeld; ++k)
          if (g0 + k < g1) put(held[k], sh.slots[g0 + k]);
        for (int g = g0 + kHeld; g < g1; ++g) put(r.at(sh.slots[g] * kSlot + lane), sh.slots[g]);
      }
      __syncthreads();
    }

    // the cut: histograms of what is left between two values, in memory until it fits the list, then there
    const int chunk = (a.slots + kPickWaves - 1) / kPickWaves;  // slots of a wavefront, where the row is searched in memory
    const int c0 = min(wave * chunk, a.slots), c1 = min(c0 + chunk, a.slots);
    if (!cut.open()) {
      float low = -FLT_MAX, high = FLT_MAX;
      bool in_list = listed;
      int in_n = n;
      int above = 0;
      double above_mass = 0.0;
      const int scale = 62 - (32 - __clz(a.V));  // (V weights of at most 1 stay below 2^63)
      const double unit = ldexp(1.0, -scale), per_unit = ldexp(1.0, scale);
      Buckets fine = rough;
      if (in_list) fine.per_unit *= kBuckets / (bound + 1.0);
      // f(z, i) for every entry between low and high, any order
      const auto each = [&](auto&& f) {
        if (in_list) {
          for (int k = tid; k < in_n; k += kPickThreads) {
            const float z = sh.list_z[k];
            if (z >= low && z <= high) f(z, sh.list_i[k]);
          }
        } else {
#pragma unroll 4
          for (int s = c0; s < c1; ++s) {
            const float z = r.at(s * kSlot + lane);
            if (z > -INFINITY && z >= low && z <= high) f(z, s * kSlot + lane);
          }
        }
      };
      for (bool inside = false;; inside = true) {
        __syncthreads();
        if (tid < kBuckets) {
          sh.count[tid] = 0;
          sh.mass[tid] = 0;
        }
        __syncthreads();
        each([&](float z, int) {
          const int b = fine.of(z);
          atomicAdd(&sh.count[b], 1u);
          if (cut.mass < INFINITY) atomicAdd(&sh.mass[b], static_cast<unsigned long long>(fma(weight(z, m, w.octaves), per_unit, 0.5)));
        });
        __syncthreads();
        if (wave == 0) find_bucket(sh, cut, above, above_mass, unit, inside);
        __syncthreads();
        const int b = sh.bucket;
        if (b == kBuckets) break;  // everything is kept
        const int count = sh.bucket_count;
        above = sh.at;
        above_mass = sh.above_mass;
        // the bucket's own entries: the least and the largest
        float least = INFINITY, most = -INFINITY;
        each([&](float z, int) {
          if (fine.of(z) == b) {
            least = fminf(least, z);
            most = fmaxf(most, z);
          }
        });
        low = block_all(least, fmin_op, sh.f);
        high = block_all(most, fmax_op, sh.f2);
        if (low == high || count <= kLast) {
          // a few of them, or equal ones: by index
          const bool equal = low == high;
          const int want = equal ? equal_ones(cut, above, above_mass, count, weight(low, m, w.octaves)) : count;
          int have = 0;
          const int k0 = min(tid * ((in_n + kPickThreads - 1) / kPickThreads), in_n), k1 = min(k0 + (in_n + kPickThreads - 1) / kPickThreads, in_n);
          if (in_list) {
            for (int k = k0; k < k1; ++k) have += sh.list_z[k] >= low && sh.list_z[k] <= high;
          } else {
            for (int s = c0; s < c1; ++s) {
              const float z = r.at(s * kSlot + lane);
              have += __popcll(__ballot(z >= low && z <= high));
            }
            if (lane != 0) have = 0;
          }
          int sum;
          int before = block_before(have, sh.i, &sum);
          const auto take = [&](float z, int i, int place) {
            if (equal) {
              if (place == want - 1) {
                sh.cut_z = z;
                sh.cut_i = i;
              }
            } else if (place < kLast) {
              sh.last_z[place] = z;
              sh.last_i[place] = i;
            }
          };
          if (in_list) {
            for (int k = k0; k < k1; ++k)
              if (sh.list_z[k] >= low && sh.list_z[k] <= high) take(sh.list_z[k], sh.list_i[k], before++);
          } else {
            before = __builtin_amdgcn_readfirstlane(before);
            for (int s = c0; s < c1; ++s) {
              const float z = r.at(s * kSlot + lane);
              const bool is = z >= low && z <= high;
              const uint64_t hit = __ballot(is);
              if (is) take(z, s * kSlot + lane, before + __popcll(hit & ((1ull << lane) - 1)));
              before += __popcll(hit);
            }
          }
          __syncthreads();
          if (!equal && wave == 0) {
            const float z = lane < count ? sh.last_z[lane] : -INFINITY;
            const double e = weight(z, m, w.octaves);
            int rank = 0;
            double ahead = 0.0;
            for (int j = 0; j < count; ++j) {
              const float zj = __shfl(z, j, 64);
              const double ej = __shfl(e, j, 64);
              if (zj > z || (zj == z && j < lane)) {
                ++rank;
                ahead += ej;
              }
            }
            const bool hit = lane < count && cut.reached(static_cast<int64_t>(above) + rank + 1, above_mass + ahead + e);
            const int end = wave_reduce_dpp(hit ? rank : count - 1, [](int x, int y) { return min(x, y); });
            if (lane < count && rank == end) {
              sh.cut_z = z;
              sh.cut_i = sh.last_i[lane];
            }
          }
          __syncthreads();
          found = {sh.cut_z, sh.cut_i};
          break;
        }
        if (!in_list && !listed && count <= kList) {
          // they fit the list now
          int have = 0;
          for (int s = c0; s < c1; ++s) {
            const float z = r.at(s * kSlot + lane);
            have += __popcll(__ballot(z >= low && z <= high));
          }
          if (lane != 0) have = 0;
          int sum;
          int before = __builtin_amdgcn_readfirstlane(block_before(have, sh.i, &sum));
          for (int s = c0; s < c1; ++s) {
            const float z = r.at(s * kSlot + lane);
            const bool is = z >= low && z <= high;
            const uint64_t hit = __ballot(is);
            if (is) {
              const int to = before + __popcll(hit & ((1ull << lane) - 1));
              sh.list_z[to] = z;
              sh.list_i[to] = s * kSlot + lane;
            }
            before += __popcll(hit);
          }
          in_list = true;
          in_n = count;
        }
        fine = buckets_of(high, static_cast<double>(high) - static_cast<double>(low));
      }
    }

    if (!listed) {
      // the kept entries' sums slot by slot, in place of the slots' own
      for (int s = c0; s < c1; ++s) {
        const float z = r.at(s * kSlot + lane);
        const double e = weight(z, m, w.octaves);
        const double sum = wave_sum_d(found.keeps(z, s * kSlot + lane) && likely(e) ? e : 0.0);
        if (lane == 0) slot_sum[s] = sum;
      }
      __syncthreads();
      mine = 0.0;
      for (int s = s0; s < s1; ++s) mine += slot_sum[s];
    }
  }

  if (listed) {
    // a thread has up to kList / kPickThreads neighbours of the list
    constexpr int kMine = kList / kPickThreads;
    const int q = (n + kPickThreads - 1) / kPickThreads;
    double e[kMine];
    mine = 0.0;
#pragma unroll
    for (int j = 0; j < kMine; ++j) {
      e[j] = 0.0;
      const int k = tid * q + j;
      if (j < q && k < n) {
        const float z = sh.list_z[k];
        const double v = weight(z, m, w.octaves);
        if (found.keeps(z, sh.list_i[k]) && likely(v)) e[j] = v;
      }
      mine += e[j];
    }
    double kept;
    const double before = block_before(mine, sh.d, &kept);
    const double target = w.u * kept;
    // (the largest entry is kept: some thread has a share)
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
    return;
  }

  // by the slots' sums: the slot, then its entry
  const bool raw = w.free();
  const auto share = [&](int s) { return raw ? slot_sum[s] * weight(slot_max[s], m, w.octaves) : slot_sum[s]; };
  double kept;
  const double before = block_before(mine, sh.d, &kept);
  const double target = w.u * kept;
  int owner = block_min(mine > 0.0 && before + mine > target ? tid : INT_MAX, sh.i);
  if (owner == INT_MAX) owner = -block_min(mine > 0.0 ? -tid : 0, sh.i);
  if (tid == owner) {
    double upto = before;
    int pick = -1, last = s0;
    double pick_before = before, last_before = before;
    for (int s = s0; s < s1; ++s) {
      const double e = share(s);
      if (e > 0.0) {
        last = s;
        last_before = upto;
        if (pick < 0 && upto + e > target) {
          pick = s;
          pick_before = upto;
        }
      }
      upto += e;
    }
    sh.slot = pick < 0 ? last : pick;
    sh.before = pick < 0 ? last_before : pick_before;
  }
  __syncthreads();
  const int slot = sh.slot;
  double others = 0.0;
  for (int s = s0; s < s1; ++s)
    if (s != slot) others += share(s);
  others = block_sum_d(others, sh.d2);
  if (wave == 0) {
    const float z = r.at(slot * kSlot + lane);
    double e = weight(z, m, w.octaves);
    if (!raw && !(found.keeps(z, slot * kSlot + lane) && likely(e))) e = 0.0;
    const double upto = sh.before + wave_upto(e);
    const uint64_t has = __ballot(e > 0.0), hit = __ballot(e > 0.0 && upto > target);
    const int at = hit ? __ffsll(static_cast<unsigned long long>(hit)) - 1 : 63 - __clzll(static_cast<long long>(has));
    others += wave_sum_d(lane == at ? 0.0 : e);
    if (lane == at) answer(slot * kSlot + at, static_cast<float>(-log1p(others / e)));
  }
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
}

size_t draw_bytes(int rows, int V) {
  const size_t slots = static_cast<size_t>(rows) * ceil_div(V, kSlot);
  return (slots * 12 + 15) / 16 * 16;
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
  const DrawArgs a = {logits, ld, V, slots, logit_rows, static_cast<const int*>(source), static_cast<const float*>(temperature),
                      static_cast<const int*>(top_k), static_cast<const float*>(top_p), static_cast<const float*>(min_p),
                      static_cast<const float*>(uniform), static_cast<const float*>(penalties), static_cast<int*>(token), static_cast<float*>(logprob),
                      sums, reinterpret_cast<float*>(sums + static_cast<size_t>(rows) * slots)};
  const uintptr_t wide = io == RWKV_IO_F16 ? 7 : 15;
  const bool vec = (reinterpret_cast<uintptr_t>(logits) & wide) == 0 && (ld % 4 == 0 || logit_rows == 1) &&
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
