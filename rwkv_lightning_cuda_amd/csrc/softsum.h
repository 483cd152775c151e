// What the two files of the log probabilities share: the running sums of a softmax and its entropy, the order of the alternatives, and
// the results.
#pragma once

#include "ops.h"

namespace rwkv {

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLowest = -3.402823466e38f;
constexpr float kGone = -200.0f;  // e^-200 is 0 in fp32; a difference that is multiplied by it must not be infinite

// by value, as as_half2: a bit cast of a vector's element reads element 0
__device__ __forceinline__ int as_int(float v) { return __builtin_bit_cast(int, v); }
__device__ __forceinline__ float as_float(int v) { return __builtin_bit_cast(float, v); }
template <int D>
__device__ __forceinline__ float lane_xor_f(float v) {
  return as_float(lane_xor_dpp<D>(as_int(v)));
}

// m = max z, S = sum e^(z - m), U = sum (z - m) e^(z - m) of the entries seen so far.  S is kept as n + s: n entries that are the
// largest, a 1 each, and the others, so that the logarithm of a row that is nearly sure of one entry does not lose the others beside
// the 1.  m starts at the lowest finite value, not at -infinity: differences with it are no NaN, and S stays 0 as long as every entry is
// -infinity.  A NaN or +infinity among the entries makes s a NaN that stays.
struct SoftSum {
  float m = kLowest, s = 0.0f, u = 0.0f, n = 0.0f;
  __device__ __forceinline__ SoftSum() {}
  __device__ __forceinline__ explicit SoftSum(const float4_t& v) : m(v[0]), s(v[1]), u(v[2]), n(v[3]) {}
  __device__ __forceinline__ float4_t stored() const { return float4_t{m, s, u, n}; }
  // an entry that is at most m
  __device__ __forceinline__ void add(float z) {
    const float d = z - m;
    const float p = __builtin_amdgcn_exp2f(d * kLog2e);
    s += d == 0.0f ? 0.0f : p;
    n += d == 0.0f ? 1.0f : 0.0f;
    u = fmaf(fmaxf(d, kGone), p, u);
  }
  // one that is less than m
  __device__ __forceinline__ void add_smaller(float z) {
    const float d = z - m;
    const float p = __builtin_amdgcn_exp2f(d * kLog2e);
    s += p;
    u = fmaf(fmaxf(d, kGone), p, u);
  }
  // an m that is as large or larger
  __device__ __forceinline__ void raise(float to) {
    const bool same = m == to;
    const float t = fmaxf(m - to, kGone);
    const float f = __builtin_amdgcn_exp2f(t * kLog2e);
    u = f * fmaf(t, s + n, u);
    s = same ? s : f * (s + n);
    n = same ? n : 0.0f;
    m = to;
  }
  __device__ __forceinline__ void merge(SoftSum o) {
    const float to = fmaxf(m, o.m);
    raise(to);
    o.raise(to);
    s += o.s;
    u += o.u;
    n += o.n;
  }
  // with what the lane of the other value of bit D has: both end with the same bits
  template <int D>
  __device__ __forceinline__ void merge_lanes() {
    SoftSum o;
    o.m = lane_xor_f<D>(m);
    o.s = lane_xor_f<D>(s);
    o.u = lane_xor_f<D>(u);
    o.n = lane_xor_f<D>(n);
    merge(o);
  }
  __device__ __forceinline__ void merge_wave() {  // the largest first: one exponential instead of twelve in a row
    const float to = wave_reduce_dpp(m, [](float x, float y) { return fmaxf(x, y); });
    raise(to);
    s = wave_sum_dpp(s);
    u = wave_sum_dpp(u);
    n = wave_sum_dpp(n);
  }
  __device__ __forceinline__ bool empty() const { return n + s == 0.0f; }
  // ln(n + s); with n = 1 what the sum has lost of s is made good: ln(1 + s) = ln(w) s / (w - 1) for the rounded w = 1 + s
  __device__ __forceinline__ float log_sum() const {
    const float w = n + s;
    const float l = logf(w);
    return n != 1.0f ? l : w == 1.0f ? s : w < 2.0f ? l * (s / (w - 1.0f)) : l;
  }
};

// log probability and entropy of a row: ln S - U / S is a sum of two terms that are not negative, nothing cancels.  token_logit is
// that of the row's token, looked at only where it is an entry.
__device__ __forceinline__ void write_logprobs(const SoftSum& a, const TokenLogprobs& out, int64_t row, int V, int token, float token_logit) {
  const float log_s = a.log_sum();
  if (out.logprob) out.logprob[row] = token < 0 ? 0.0f : token >= V ? __builtin_nanf("") : a.empty() ? -INFINITY : token_logit - a.m - log_s;
  if (out.entropy) out.entropy[row] = a.empty() ? 0.0f : log_s - a.u / (a.n + a.s);
}

// The order "larger first, equal ones by index" as that of whole numbers: the value's bits made to rise with it above the index's
// complement.  No entry has the key 0.  (-0 is 0; NaN has no place and must not come here.)
typedef unsigned long long key_t;
__device__ __forceinline__ uint32_t rising(float z) {
  const uint32_t b = __builtin_bit_cast(uint32_t, z + 0.0f);
  return b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u);
}
__device__ __forceinline__ key_t key_of(float z, int i) { return static_cast<key_t>(rising(z)) << 32 | ~static_cast<uint32_t>(i); }
__device__ __forceinline__ float key_value(key_t k) {
  const uint32_t b = static_cast<uint32_t>(k >> 32);
  return __builtin_bit_cast(float, b & 0x80000000u ? b ^ 0x80000000u : ~b);
}
__device__ __forceinline__ int key_index(key_t k) { return static_cast<int>(~static_cast<uint32_t>(k)); }

constexpr int kCandidates = 1024;

// Entries that may be among the first top_n, in LDS.  They come in the order of an atomic counter, which no result depends on.
template <int NT>
struct Candidates {
  key_t list[2][kCandidates];
  float group_max[256];
  int n;
};

// A value that the top_n-th largest of the wavefront's N values per lane reaches: that value with its last 16 bits cut off (downwards: a
// bound may be loose by 2^-7), found bit by bit from the first.  (16 counts of a ballot: 0.7 us for a block's first bound; counting for each
// of its values how many are larger took 3.2.)  -infinity where there are not as many; NaN counts as that.
template <int N>
__device__ __forceinline__ float wave_bound(const float (&v)[N], int top_n) {
  uint32_t r[N];
#pragma unroll
  for (int i = 0; i < N; ++i) r[i] = v[i] == v[i] ? rising(v[i]) : 0u;
  uint32_t found = 0;
#pragma unroll
  for (int bit = 31; bit >= 16; --bit) {
    const uint32_t next = found | 1u << bit;
    int count = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) count += __builtin_popcountll(__ballot(r[i] >= next));
    if (count >= top_n) found = next;
  }
  constexpr uint32_t kOfInfinity = 0x007fffffu;  // rising(-infinity)
  return found <= kOfInfinity ? -INFINITY : __builtin_bit_cast(float, found & 0x80000000u ? found ^ 0x80000000u : ~found);
}

// The same of the maxima of 64 or 256 groups of threads: top_n entries are at least as large, so that none below it is among the first
// top_n.  Every thread of the block comes here; every wavefront finds the same.
template <int NT>
__device__ __forceinline__ float first_bound(Candidates<NT>& c, int top_n, float mine) {
  static_assert(NT == 256, "four threads to one of 64 groups");
  const int tid = threadIdx.x, lane = threadIdx.x & 63;
  if (top_n <= 24) {
    if (mine != mine) mine = -INFINITY;
    mine = fmaxf(mine, lane_xor_f<1>(mine));
    mine = fmaxf(mine, lane_xor_f<2>(mine));
    if ((tid & 3) == 0) c.group_max[tid >> 2] = mine;
    __syncthreads();
    const float v[1] = {c.group_max[lane]};
    return wave_bound(v, top_n);
  }
  c.group_max[tid] = mine;
  __syncthreads();
  const float v[4] = {c.group_max[lane], c.group_max[64 + lane], c.group_max[128 + lane], c.group_max[192 + lane]};
  return wave_bound(v, top_n);
}

// The first top_n of the n in list `from`, in order, to the other list.  Behind a barrier; the caller waits for what it writes.
template <int NT>
__device__ __forceinline__ void thin_out(Candidates<NT>& c, int from, int n, int top_n) {
  const key_t* list = c.list[from];
  for (int k = threadIdx.x; k < n; k += NT) {
    const key_t mine = list[k];
    int before = 0;
#pragma unroll 8
    for (int i = 0; i < n; ++i) before += list[i] > mine;
    if (before < top_n) c.list[from ^ 1][before] = mine;
  }
}

template <int NT>
__device__ __forceinline__ void offer(Candidates<NT>& c, int to, key_t key) {
  const int at = atomicAdd(&c.n, 1);
  if (at < kCandidates) c.list[to][at] = key;
}

// key 0: none
__device__ __forceinline__ void write_alternative(const TokenLogprobs& out, int64_t row, int place, key_t key, float m, float log_s) {
  const int64_t o = row * out.top_n + place;
  out.top_ids[o] = key ? key_index(key) : -1;
  out.top_logprobs[o] = key ? key_value(key) - m - log_s : -INFINITY;
}

}  // namespace rwkv
