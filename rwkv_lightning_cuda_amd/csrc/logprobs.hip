// Log probabilities of given tokens from a row of logits z: what a server returns beside a sampled token and what scoring a
// text asks for.  No counterpart in the reference (its sampler keeps the probabilities to itself, src/utils/sampling.cu:205-471).
//
//   m = max z;  S = sum e^(z_i - m);  U = sum (z_i - m) e^(z_i - m)
//   log probability of t = z_t - m - ln S;  entropy = ln S - U / S (a sum of two terms that are not negative: nothing cancels)
//   rank of t = entries ahead of it in the order "larger first, equal ones by index";  alternatives = the first top_n in that order
//
// Entries of -infinity have probability 0 and are no alternatives; a row of nothing else gives log probability -infinity, entropy 0
// and no alternative.
#include "softsum.h"

namespace rwkv {

namespace {

constexpr int kCandidates = 1024;  // places for entries that may be among the first top_n
constexpr int kRefine = 4;         // batches between looks at whether the candidates can be thinned out

struct LogprobArgs {
  const void* logits;
  int64_t ld;
  int V;
  TokenLogprobs out;
};

__device__ __forceinline__ float next_above(float v) {  // the smallest float above v; NaN above +infinity
  const uint32_t b = __builtin_bit_cast(uint32_t, v);
  return v == 0.0f ? __builtin_bit_cast(float, 1u) : __builtin_bit_cast(float, v > 0.0f ? b + 1 : b - 1);
}

// One block per row, which it reads once: 64 bytes per thread at a time, the next 64 requested before they are looked at.  A thread
// keeps m, S and U of its entries and raises m when a batch exceeds it.  The rank is a count against the token's logit, which is
// read first.  Alternatives: of the first batch the largest entry of each of 64 or 256 groups of threads is known; top_n of these are
// at least as large as the top_n-th of them, so that nothing below it can be an alternative.  What is not below goes to a list in LDS (its
// order is that of an atomic counter, its use is not), which is sorted by counting at the end, and thinned out to the first top_n - with
// the last one as the new bound - whenever it has grown to four times as many.  A list that overflows (a row that rises, or is of one
// value) is given up: the alternatives are then found one after the other in top_n walks over the row.
template <typename T, int NT>
__global__ __launch_bounds__(NT) void token_logprobs_kernel(LogprobArgs a) {
  constexpr int VE = 16 / sizeof(T);  // entries of a 16-byte vector
  constexpr int VB = 4;               // vectors of a batch
  typedef T vec_t __attribute__((ext_vector_type(VE)));
  __shared__ float cand_z[2][kCandidates];
  __shared__ int cand_i[2][kCandidates];
  __shared__ __align__(16) float group_max[256];
  __shared__ float red[4][NT / 64];
  __shared__ int n_cand;
  __shared__ float bound_s;
  const int tid = threadIdx.x;
  const T* z = static_cast<const T*>(a.logits) + blockIdx.x * a.ld;
  const int V = a.V, top_n = a.out.top_n;
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
        next[q] = body[v];
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
  const int t = a.out.tokens ? a.out.tokens[blockIdx.x] : -1;
  const bool has_token = t >= 0 && t < V;
  const float zt = has_token ? static_cast<float>(z[t]) : 0.0f;
  const bool count = a.out.rank && has_token;
  const float zt_above = next_above(zt);
  if (top_n > 0 && tid == 0) n_cand = 0;

  SoftSum sum;
  int ahead = 0;
  float bound = INFINITY;
  int list = 0;
  auto offer = [&](float v, int i) {
    if (v >= bound && v > -INFINITY) {
      const int at = atomicAdd(&n_cand, 1);
      if (at < kCandidates) {
        cand_z[list][at] = v;
        cand_i[list][at] = i;
      }
    }
  };
  // the top_n-th largest of the groups' maxima (equal ones by group): every thread of the block comes here
  auto first_bound = [&](float mine) {
    const int groups = top_n <= 24 ? 64 : 256;
    if (mine != mine) mine = -INFINITY;
    const int width = NT / groups;
    if (width > 1) mine = fmaxf(mine, __builtin_bit_cast(float, lane_xor_dpp<1>(__builtin_bit_cast(int, mine))));
    if (width > 2) mine = fmaxf(mine, __builtin_bit_cast(float, lane_xor_dpp<2>(__builtin_bit_cast(int, mine))));
    if (width > 4) mine = fmaxf(mine, __builtin_bit_cast(float, lane_xor_dpp<4>(__builtin_bit_cast(int, mine))));
    if (width > 8) mine = fmaxf(mine, __builtin_bit_cast(float, lane_xor_dpp<8>(__builtin_bit_cast(int, mine))));
    if (tid % width == 0) group_max[tid / width] = mine;
    __syncthreads();
    if (tid < groups) {
      const float v = group_max[tid];
      int before = 0;
      for (int i = 0; i < groups; i += 4) {
        const float4_t w = *reinterpret_cast<const float4_t*>(group_max + i);
#pragma unroll
        for (int e = 0; e < 4; ++e) before += ahead_of(w[e], i + e, v, tid);
      }
      if (before == top_n - 1) bound_s = v;
    }
    __syncthreads();
    bound = bound_s;
  };
  // the first top_n of the list, in order, to the other list; returns how many there were
  auto thin_out = [&](int n) {
    for (int c = tid; c < n; c += NT) {
      const float v = cand_z[list][c];
      const int i = cand_i[list][c];
      int before = 0;
      for (int k = 0; k < n; ++k) before += ahead_of(cand_z[list][k], cand_i[list][k], v, i);
      if (before < top_n) {
        cand_z[list ^ 1][before] = v;
        cand_i[list ^ 1][before] = i;
      }
    }
    list ^= 1;
  };

  // (fmaxf of a NaN and a number is the number)
  for (int b = 0; b < batches || b == 0; ++b) {
    float x[VB * VE];
#pragma unroll
    for (int q = 0; q < VB; ++q)
#pragma unroll
      for (int e = 0; e < VE; ++e) x[q * VE + e] = static_cast<float>(next[q][e]);
    if (b + 1 < batches) request(b + 1);
    float most = fmaxf(x[0], x[1]);
#pragma unroll
    for (int e = 2; e < VB * VE; ++e) most = fmaxf(most, x[e]);
    if (top_n > 0) {
      if (b == 0) {
        first_bound(fmaxf(most, stray_z));
        offer(stray_z, stray);
      }
      if (most >= bound) {
        uint32_t mask = 0;
#pragma unroll
        for (int e = VB * VE - 1; e >= 0; --e) mask = mask * 2 + (x[e] >= bound);
        while (mask) {
          const int e = __builtin_ctz(mask);
          mask &= mask - 1;
          const int i = head + ((b * VB + e / VE) * NT + tid) * VE + e % VE;
          if (i < tail) offer(static_cast<float>(z[i]), i);  // (again from memory: a register cannot be chosen by a number)
        }
      }
      if (b % kRefine == kRefine - 1) {
        __syncthreads();
        const int n = n_cand;
        if (n > 4 * top_n && n <= kCandidates) {
          thin_out(n);
          __syncthreads();
          bound = cand_z[list][top_n - 1];
          if (tid == 0) n_cand = top_n;
        }
        __syncthreads();
      }
    }
    if (count) {
      // entries ahead of the token: as large in front of it, larger behind it (the vector it lies in: larger, made good at the end)
#pragma unroll
      for (int q = 0; q < VB; ++q) {
        const float least = head + ((b * VB + q) * NT + tid) * VE + VE <= t ? zt : zt_above;
#pragma unroll
        for (int e = 0; e < VE; ++e) ahead += x[q * VE + e] >= least;
      }
    }
    if (most > sum.m) sum.raise(most);
#pragma unroll
    for (int e = 0; e < VB * VE; ++e) {
      const float d = x[e] - sum.m;
      const float p = __builtin_amdgcn_exp2f(d * kLog2e);
      sum.s += p;
      sum.u = fmaf(fmaxf(d, kGone), p, sum.u);
    }
  }
  {
    if (stray_z > sum.m) sum.raise(stray_z);
    const float d = stray_z - sum.m;
    const float p = __builtin_amdgcn_exp2f(d * kLog2e);
    sum.s += p;
    sum.u = fmaf(fmaxf(d, kGone), p, sum.u);
    if (count) ahead += stray < V && ahead_of(stray_z, stray, zt, t);
    // equal entries of the token's own vector in front of it
    if (count && tid == 0 && t >= head && t < tail)
      for (int i = t - (t - head) % VE; i < t; ++i) ahead += static_cast<float>(z[i]) == zt;
  }

  // the block's sums
  {
    const float m = wave_reduce_dpp(sum.m, [](float x, float y) { return fmaxf(x, y); });
    if ((tid & 63) == 0) red[0][tid >> 6] = m;
    __syncthreads();
    float all = red[0][0];
#pragma unroll
    for (int i = 1; i < NT / 64; ++i) all = fmaxf(all, red[0][i]);
    sum.raise(all);
    const float s = wave_sum_dpp(sum.s), u = wave_sum_dpp(sum.u);
    const int c = wave_reduce_dpp(ahead, [](int x, int y) { return x + y; });
    if ((tid & 63) == 0) {
      red[1][tid >> 6] = s;
      red[2][tid >> 6] = u;
      red[3][tid >> 6] = __builtin_bit_cast(float, c);
    }
    __syncthreads();
    sum.s = sum.u = 0.0f;
    ahead = 0;
#pragma unroll
    for (int i = 0; i < NT / 64; ++i) {
      sum.s += red[1][i];
      sum.u += red[2][i];
      ahead += __builtin_bit_cast(int, red[3][i]);
    }
  }
  const float log_s = logf(sum.s);
  if (tid == 0) {
    write_logprobs(sum, a.out, blockIdx.x, V, &zt);
    if (a.out.rank) a.out.rank[blockIdx.x] = !has_token || zt != zt ? -1 : ahead;
  }
  if (top_n == 0) return;

  int* ids = a.out.top_ids + static_cast<int64_t>(blockIdx.x) * top_n;
  float* tops = a.out.top_logprobs + static_cast<int64_t>(blockIdx.x) * top_n;
  const int n = n_cand;
  if (n <= kCandidates) {
    thin_out(n);
    __syncthreads();
    if (tid < top_n) {
      const bool there = tid < n;
      ids[tid] = there ? cand_i[list][tid] : -1;
      tops[tid] = there ? cand_z[list][tid] - sum.m - log_s : -INFINITY;
    }
    return;
  }
  // one after the other: the first entry behind the one before
  float last = INFINITY;
  int last_i = -1;
  for (int k = 0; k < top_n; ++k) {
    float best = -INFINITY;
    int bi = V;
    for (int i = tid; i < V; i += NT) {
      const float v = static_cast<float>(z[i]);
      if (ahead_of(last, last_i, v, i) && v > best) {
        best = v;
        bi = i;
      }
    }
    const float wave_best = wave_reduce_dpp(best, [](float x, float y) { return fmaxf(x, y); });
    bi = wave_reduce_dpp(best == wave_best ? bi : V, [](int x, int y) { return min(x, y); });
    __syncthreads();
    if ((tid & 63) == 0) {
      cand_z[0][tid >> 6] = wave_best;
      cand_i[0][tid >> 6] = bi;
    }
    __syncthreads();
    best = -INFINITY;
    bi = V;
    for (int i = 0; i < NT / 64; ++i) {
      if (cand_i[0][i] < V && ahead_of(cand_z[0][i], cand_i[0][i], best, bi)) {
        best = cand_z[0][i];
        bi = cand_i[0][i];
      }
    }
    if (tid == 0) {
      ids[k] = bi < V ? bi : -1;
      tops[k] = bi < V ? best - sum.m - log_s : -INFINITY;
    }
    last = best;
    last_i = bi;
  }
}

template <typename T>
void launch_rows(hipStream_t st, int rows, const LogprobArgs& a) {
  if (rows <= 2 * device_cu_count()) hipLaunchKernelGGL((token_logprobs_kernel<T, 1024>), dim3(rows), dim3(1024), 0, st, a);
  else hipLaunchKernelGGL((token_logprobs_kernel<T, 256>), dim3(rows), dim3(256), 0, st, a);
}

}  // namespace

size_t token_logprobs_workspace_bytes(int rows, int V, int top_n) { return 0; }

int token_logprobs_launch(hipStream_t st, int rows, int V, int io, const void* logits, int64_t ld, const TokenLogprobs& out, void* workspace) {
  LogprobArgs a = {logits, ld, V, out};
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
  const size_t need = token_logprobs_workspace_bytes(rows, V, top_n);
  RWKV_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0),
               "token_logprobs: workspace of %zu bytes (aligned to 16) needed, got %zu", need, workspace_bytes);
  return token_logprobs_launch(as_stream(s), rows, V, io, logits, ld, out, workspace);
}

}  // extern "C"
