// Log probabilities of given tokens from a row of logits z: what a server returns beside a sampled token and what scoring a
// text asks for.  No counterpart in the reference (its sampler keeps the probabilities to itself, src/utils/sampling.cu:205-471).
//
//   m = max z;  S = sum e^(z_i - m);  U = sum (z_i - m) e^(z_i - m)
//   log probability of t = z_t - m - ln S;  entropy = ln S - U / S (a sum of two terms that are not negative: nothing cancels)
//   rank of t = entries ahead of it in the order "larger first, equal ones by index";  alternatives = the first top_n in that order
//
// Bound by memory where rows are many (fp32: 2048 x 65536, 537 MB, 87 us = 6.2 TB/s, non-temporal loads; fp16 80 us, there by the 14
// vector instructions per entry), by the chain of two launches and their reductions where they are few (one row with 5 alternatives 5.5 + 4 us,
// 64 rows with 20 9.9 + 5).
//
// Entries of -infinity have probability 0 and are no alternatives; a row of nothing else gives log probability -infinity, entropy 0
// and no alternative.
#include "logprobs_parts.h"
#include "softsum.h"

namespace rwkv {

namespace {

constexpr int kThreads = kLogprobThreads;
constexpr int kRefine = 4;  // batches between looks at whether the candidates can be thinned out

struct LogprobArgs {
  const void* logits;
  int64_t ld;
  int V;
  TokenLogprobs out;
  // rows in several parts: what each leaves
  int parts, part_len;
  float4_t* sums;  // [rows][parts]
  int* ahead;      // [rows][parts]: entries ahead of the token
  float* token_logit;  // [rows]
  key_t* keys;     // [rows][parts][part_keys(top_n)] in any order, 0 past the last
};

static_assert(sizeof(float4_t) == 16 && sizeof(key_t) == 8, "PartBytes");
static_assert(part_keys(kMaxAlternatives) <= 256, "written by one thread each");

__device__ __forceinline__ float next_above(float v) {  // the smallest float above v; NaN above +infinity
  const uint32_t b = __builtin_bit_cast(uint32_t, v);
  return v == 0.0f ? __builtin_bit_cast(float, 1u) : __builtin_bit_cast(float, v > 0.0f ? b + 1 : b - 1);
}

// One block per row, or per part of one, which it reads once: 64 bytes per thread at a time, the next 64 requested before they are
// looked at.  A thread keeps the sums of its entries against the largest that its wavefront has seen, which few batches raise.  The rank
// is a count against the token's logit, which is read first.  Alternatives: what is not below the bound that the first batch gives goes to
// a list in LDS, which is thinned out to the first top_n - with the last one as the new bound - whenever it has grown to four times as
// many.  A list that overflows (a row that rises, or is of one value) is given up: the alternatives are then found one after the other in
// top_n walks.
template <typename T, bool PART>
__global__ __launch_bounds__(kThreads) void token_logprobs_kernel(LogprobArgs a) {
  constexpr int NT = kThreads;
  constexpr int VE = 16 / sizeof(T);  // entries of a 16-byte vector
  constexpr int VB = 4;               // vectors of a batch
  typedef T vec_t __attribute__((ext_vector_type(VE)));
  __shared__ __align__(16) Candidates<NT> cand;
  __shared__ float4_t waves[NT / 64];
  __shared__ int waves_ahead[NT / 64];
  const int tid = threadIdx.x;
  const int top_n = a.out.top_n;
  const T* row = static_cast<const T*>(a.logits) + blockIdx.x * a.ld;
  // entries first .. first + V - 1 of the row; every index below counts from `first`
  const int first = PART ? blockIdx.y * a.part_len : 0;
  const int V = PART ? min(a.part_len, a.V - first) : a.V;
  const T* z = row + first;
  const int misaligned = static_cast<int>((reinterpret_cast<uintptr_t>(z) & 15) / sizeof(T));
  const int head = misaligned ? min(VE - misaligned, V) : 0;  // entries in front of the first 16-byte boundary
  const int vecs = (V - head) / VE;
  const int tail = head + vecs * VE;                          // first entry behind the last vector
  const vec_t* body = reinterpret_cast<const vec_t*>(z + head);
  const int batches = (vecs + NT * VB - 1) / (NT * VB);

  vec_t next[VB];
  auto request = [&](int b) {
#pragma unroll
    for (int q = 0; q < VB; ++q) {
      const int v = (b * VB + q) * NT + tid;
      if (v < vecs) {
        next[q] = __builtin_nontemporal_load(body + v);
      } else {
#pragma unroll
        for (int e = 0; e < VE; ++e) next[q][e] = static_cast<T>(-INFINITY);
      }
    }
  };
  request(0);
  // the entries of the two ends, at most one per thread
  const int stray = tid < head ? tid : tail + tid - head;
  const float stray_z = stray < V ? static_cast<float>(z[stray]) : -INFINITY;
  const int token = a.out.tokens ? a.out.tokens[blockIdx.x] : -1;
  const bool has_token = token >= 0 && token < a.V;
  const float zt = has_token ? static_cast<float>(row[token]) : 0.0f;
  const int t = token - first;  // (may lie in front of this part or behind it)
  const bool count = a.out.rank && has_token;
  const float zt_above = next_above(zt);
  if (top_n > 0 && tid == 0) cand.n = 0;

  SoftSum sum;
  int ahead = 0;
  float bound = INFINITY;
  int list = 0;
  for (int b = 0; b < batches || b == 0; ++b) {
    float x[VB * VE];
#pragma unroll
    for (int q = 0; q < VB; ++q)
#pragma unroll
      for (int e = 0; e < VE; ++e) x[q * VE + e] = static_cast<float>(next[q][e]);
    if (b + 1 < batches) request(b + 1);
    float most = fmaxf(x[0], x[1]);  // (fmaxf of a NaN and a number is the number)
#pragma unroll
    for (int e = 2; e < VB * VE; ++e) most = fmaxf(most, x[e]);
    if (top_n > 0) {
      if (b == 0) {
        bound = first_bound(cand, top_n, fmaxf(most, stray_z));
        if (stray_z >= bound && stray_z > -INFINITY) offer(cand, list, key_of(stray_z, first + stray));
      }
      if (most >= bound) {
#pragma unroll
        for (int q = 0; q < VB; ++q)
#pragma unroll
          for (int e = 0; e < VE; ++e) {
            const float v = x[q * VE + e];
            if (v >= bound && v > -INFINITY) offer(cand, list, key_of(v, first + head + ((b * VB + q) * NT + tid) * VE + e));
          }
      }
      if (b % kRefine == kRefine - 1) {
        __syncthreads();
        const int n = cand.n;
        if (n > 4 * top_n && n <= kCandidates) {
          thin_out(cand, list, n, top_n);
          list ^= 1;
          __syncthreads();
          bound = key_value(cand.list[list][top_n - 1]);
          if (tid == 0) cand.n = top_n;
        }
        __syncthreads();
      }
    }
    if (count) {
      // entries ahead of the token: as large in front of it, larger behind it (the vector it lies in: larger, made good at the end)
#pragma unroll
      for (int q = 0; q < VB; ++q) {
        const int v = (b * VB + q) * NT + tid;
        const float least = v < vecs && head + v * VE + VE <= t ? zt : zt_above;
#pragma unroll
        for (int e = 0; e < VE; ++e) ahead += x[q * VE + e] >= least;
      }
    }
    if (__any(most >= sum.m)) {  // (m is the wavefront's: one decision, and few batches come here)
      sum.raise(fmaxf(sum.m, wave_reduce_dpp(most, [](float v, float w) { return fmaxf(v, w); })));
#pragma unroll
      for (int e = 0; e < VB * VE; ++e) sum.add(x[e]);
    } else {
#pragma unroll
      for (int e = 0; e < VB * VE; ++e) sum.add_smaller(x[e]);
    }
  }
  if (head > 0 || tail < V) {
    const float to = wave_reduce_dpp(stray_z, [](float v, float w) { return fmaxf(v, w); });
    sum.raise(fmaxf(sum.m, to));
    sum.add(stray_z);
    if (count) ahead += stray < V && (stray_z > zt || (stray_z == zt && stray < t));
  }
  // equal entries of the token's own vector in front of it
  if (count && tid == 0 && t >= head && t < tail)
    for (int i = t - (t - head) % VE; i < t; ++i) ahead += static_cast<float>(z[i]) == zt;

  // the block's sums
  sum.merge_wave();
  ahead = wave_reduce_dpp(ahead, [](int x, int y) { return x + y; });
  if ((tid & 63) == 0) {
    waves[tid >> 6] = sum.stored();
    waves_ahead[tid >> 6] = ahead;
  }
  __syncthreads();
  sum = SoftSum();
  ahead = 0;
#pragma unroll
  for (int i = 0; i < NT / 64; ++i) {
    sum.merge(SoftSum(waves[i]));
    ahead += waves_ahead[i];
  }
  const int64_t at = static_cast<int64_t>(blockIdx.x) * a.parts + blockIdx.y;
  float log_s = 0.0f;
  if constexpr (PART) {
    if (tid == 0) {
      a.sums[at] = sum.stored();
      a.ahead[at] = ahead;
      if (blockIdx.y == 0) a.token_logit[blockIdx.x] = zt;
    }
  } else if (tid < 64) {
    log_s = sum.log_sum();
    if (tid == 0) {
      write_logprobs(sum, a.out, blockIdx.x, V, token, zt);
      if (a.out.rank) a.out.rank[blockIdx.x] = !has_token || zt != zt ? -1 : ahead;
    }
  }
  if (top_n == 0) return;
  static_assert(kMaxAlternatives <= 64, "one wavefront writes them");
  const int slots = part_keys(top_n);
  auto write = [&](int place, key_t key) {
    if constexpr (PART) a.keys[at * slots + place] = key;
    else write_alternative(a.out, blockIdx.x, place, key, sum.m, log_s);
  };

  const int n = cand.n;
  if (PART && n <= slots) {
    if (tid < slots) write(tid, tid < n ? cand.list[list][tid] : 0);
    return;
  }
  if (PART && tid >= top_n && tid < slots) write(tid, 0);
  if (n <= kCandidates) {
    thin_out(cand, list, n, top_n);
    __syncthreads();
    if (tid < top_n) write(tid, tid < n ? cand.list[list ^ 1][tid] : 0);
    return;
  }
  // one after the other: the first entry behind the one before
  key_t last = ~static_cast<key_t>(0);
  key_t* best_of = cand.list[0];
  for (int k = 0; k < top_n; ++k) {
    key_t best = 0;
    for (int i = tid; i < V; i += NT) {
      const float v = static_cast<float>(z[i]);
      if (!(v > -INFINITY)) continue;
      const key_t key = key_of(v, first + i);
      if (key < last && key > best) best = key;
    }
    __syncthreads();
    best_of[tid] = best;
    __syncthreads();
    for (int step = NT / 2; step > 0; step /= 2) {
      if (tid < step && best_of[tid + step] > best_of[tid]) best_of[tid] = best_of[tid + step];
      __syncthreads();
    }
    last = best_of[0];
    if (tid == 0) write(k, last);
  }
}

// A block per row over what its parts have left.  Of many keys a bound is made first, as of the entries of a row.
__global__ __launch_bounds__(kThreads) void token_logprobs_join_kernel(LogprobArgs a) {
  __shared__ __align__(16) Candidates<kThreads> cand;
  __shared__ float4_t waves[kThreads / 64];
  __shared__ int waves_ahead[kThreads / 64];
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.x;
  const int top_n = a.out.top_n;
  const int total = a.parts * part_keys(top_n);
  const key_t* keys = a.keys + row * total;
  // everything that most calls need, requested at once
  const key_t own = tid < total ? keys[tid] : 0;
  const int token = a.out.tokens ? a.out.tokens[row] : -1;
  const float zt = a.token_logit[row];
  SoftSum sum;
  int ahead = 0;
  if (tid < a.parts) {
    sum = SoftSum(a.sums[row * a.parts + tid]);
    ahead = a.ahead[row * a.parts + tid];
  }
  sum.merge_wave();
  ahead = wave_reduce_dpp(ahead, [](int x, int y) { return x + y; });
  if ((tid & 63) == 0) {
    waves[tid >> 6] = sum.stored();
    waves_ahead[tid >> 6] = ahead;
  }
  if (tid == 0) cand.n = 0;
  __syncthreads();
  sum = SoftSum();
  ahead = 0;
#pragma unroll
  for (int i = 0; i < kThreads / 64; ++i) {
    sum.merge(SoftSum(waves[i]));
    ahead += waves_ahead[i];
  }
  if (tid == 0) {
    write_logprobs(sum, a.out, row, a.V, token, zt);
    if (a.out.rank) a.out.rank[row] = token < 0 || token >= a.V || zt != zt ? -1 : ahead;
  }
  if (top_n == 0) return;
  float bound = -INFINITY;
  if (total > 32) {
    float most = own ? key_value(own) : -INFINITY;
    for (int k = tid + kThreads; k < total; k += kThreads)
      if (keys[k]) most = fmaxf(most, key_value(keys[k]));
    bound = first_bound(cand, top_n, most);
  }
  if (own && key_value(own) >= bound) offer(cand, 0, own);
  for (int k = tid + kThreads; k < total; k += kThreads)
    if (keys[k] && key_value(keys[k]) >= bound) offer(cand, 0, keys[k]);
  __syncthreads();
  const int n = cand.n;
  const float log_s = sum.log_sum();
  if (n <= kCandidates) {
    thin_out(cand, 0, n, top_n);
    __syncthreads();
    if (tid < top_n) write_alternative(a.out, row, tid, tid < n ? cand.list[1][tid] : 0, sum.m, log_s);
    return;
  }
  // (equal values all over) one after the other, out of memory
  key_t last = ~static_cast<key_t>(0);
  key_t* best_of = cand.list[0];
  for (int place = 0; place < top_n; ++place) {
    key_t best = 0;
    for (int k = tid; k < total; k += kThreads)
      if (keys[k] < last && keys[k] > best) best = keys[k];
    __syncthreads();
    best_of[tid] = best;
    __syncthreads();
    for (int step = kThreads / 2; step > 0; step /= 2) {
      if (tid < step && best_of[tid + step] > best_of[tid]) best_of[tid] = best_of[tid + step];
      __syncthreads();
    }
    last = best_of[0];
    if (tid == 0) write_alternative(a.out, row, place, last, sum.m, log_s);
  }
}

template <typename T>
void launch_rows(hipStream_t st, int rows, const LogprobArgs& a) {
  if (a.parts == 1) {
    hipLaunchKernelGGL((token_logprobs_kernel<T, false>), dim3(rows), dim3(kThreads), 0, st, a);
  } else {
    hipLaunchKernelGGL((token_logprobs_kernel<T, true>), dim3(rows, a.parts), dim3(kThreads), 0, st, a);
    hipLaunchKernelGGL(token_logprobs_join_kernel, dim3(rows), dim3(kThreads), 0, st, a);
  }
}

}  // namespace

size_t token_logprobs_workspace_bytes(int rows, int V, int top_n) { return most_logprob_bytes(rows, V, top_n, device_cu_count()); }

int token_logprobs_launch(hipStream_t st, int rows, int V, int io, const void* logits, int64_t ld, const TokenLogprobs& out, void* workspace,
                          size_t workspace_bytes) {
  const size_t need = logprob_bytes(rows, V, out.top_n, device_cu_count());
  RWKV_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0),
               "token_logprobs: workspace of %zu bytes (aligned to 16) needed, got %zu", need, workspace_bytes);
  const int parts = logprob_parts(rows, V, io, device_cu_count());
  // (a multiple of a vector, so that the parts of an aligned row are aligned)
  const PartBytes p = part_bytes(rows, parts, out.top_n);
  char* ws = static_cast<char*>(workspace);
  LogprobArgs a = {logits, ld, V, out, parts, ceil_div(ceil_div(V, parts), 64) * 64, reinterpret_cast<float4_t*>(ws),
                   reinterpret_cast<int*>(ws + p.sums), reinterpret_cast<float*>(ws + p.sums + p.ahead),
                   reinterpret_cast<key_t*>(ws + p.sums + p.ahead + p.token_logit)};
  a.parts = ceil_div(V, a.part_len);  // (rounding up may leave the last one without entries)
  if (io == RWKV_IO_F16) launch_rows<half_t>(st, rows, a);
  else launch_rows<float>(st, rows, a);
  RWKV_LAUNCH_CHECK();
  return RWKV_OK;
}

int check_token_logprobs(const char* who, const TokenLogprobs& out) {
  RWKV_REQUIRE(out.top_n >= 0 && out.top_n <= kMaxAlternatives, "%s: top_n must lie in 0 .. %d, got %d", who, kMaxAlternatives, out.top_n);
  RWKV_REQUIRE(out.top_n == 0 || (out.top_ids && out.top_logprobs), "%s: top_n without its two outputs", who);
  RWKV_REQUIRE(out.tokens || (!out.logprob && !out.rank), "%s: logprob and rank need tokens", who);
  RWKV_REQUIRE(out.logprob || out.entropy || out.rank || out.top_n > 0, "%s: no output is asked for", who);
  for (const void* p : {static_cast<const void*>(out.tokens), static_cast<const void*>(out.logprob), static_cast<const void*>(out.entropy),
                        static_cast<const void*>(out.rank), static_cast<const void*>(out.top_ids), static_cast<const void*>(out.top_logprobs)})
    RWKV_REQUIRE((reinterpret_cast<uintptr_t>(p) & 3) == 0, "%s: 32-bit tensors must be aligned to 4 bytes", who);
  return RWKV_OK;
}

}  // namespace rwkv

using namespace rwkv;

extern "C" {

int rwkv_hip_token_logprobs_workspace(int rows, int V, int top_n, size_t* bytes) {
  RWKV_REQUIRE(bytes && rows > 0 && V > 0 && V <= kMaxLogprobVocab, "token_logprobs_workspace: bad arguments");
  RWKV_REQUIRE(top_n >= 0 && top_n <= kMaxAlternatives, "token_logprobs_workspace: top_n must lie in 0 .. %d, got %d", kMaxAlternatives, top_n);
  *bytes = token_logprobs_workspace_bytes(rows, V, top_n);
  return RWKV_OK;
}

int rwkv_hip_token_logprobs(rwkv_stream_t s, int rows, int V, int io, const void* logits, int64_t ld, const void* tokens, int top_n,
                            void* logprob, void* entropy, void* rank, void* top_ids, void* top_logprobs, void* workspace,
                            size_t workspace_bytes) {
  RWKV_REQUIRE(rows > 0, "token_logprobs: rows must be positive, got %d", rows);
  RWKV_REQUIRE(V > 0 && V <= kMaxLogprobVocab, "token_logprobs: V must lie in 1 .. %d, got %d", kMaxLogprobVocab, V);
  RWKV_REQUIRE(io == RWKV_IO_F16 || io == RWKV_IO_F32, "token_logprobs: unknown element type %d", io);
  RWKV_REQUIRE(logits, "token_logprobs: NULL logits");
  RWKV_REQUIRE(ld >= V, "token_logprobs: rows of %d entries lie %lld apart", V, static_cast<long long>(ld));
  RWKV_REQUIRE((reinterpret_cast<uintptr_t>(logits) & (io == RWKV_IO_F16 ? 1 : 3)) == 0, "token_logprobs: misaligned logits");
  const TokenLogprobs out = {static_cast<const int*>(tokens), top_n, static_cast<float*>(logprob), static_cast<float*>(entropy),
                             static_cast<int*>(rank), static_cast<int*>(top_ids), static_cast<float*>(top_logprobs)};
  const int rc = check_token_logprobs("token_logprobs", out);
  if (rc != RWKV_OK) return rc;
  return token_logprobs_launch(as_stream(s), rows, V, io, logits, ld, out, workspace, workspace_bytes);
}

}  // extern "C"
