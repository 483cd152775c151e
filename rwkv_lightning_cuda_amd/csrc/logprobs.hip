// Log probabilities of given tokens from a row of logits z: what a server returns beside a sampled token and what scoring a
// text asks for.  No counterpart in the reference (its sampler keeps the probabilities to itself, src/utils/sampling.cu:205-471).
//
//   m = max z;  S = sum e^(z_i - m);  U = sum (z_i - m) e^(z_i - m)
//   log probability of t = z_t - m - ln S;  entropy = ln S - U / S (a sum of two terms that are not negative: nothing cancels)
//   rank of t = entries ahead of it in the order "larger first, equal ones by index";  alternatives = the first top_n in that order
//
// Entries of -infinity have probability 0 and are no alternatives; a row of nothing else gives log probability -infinity, entropy 0
// and no alternative.
#include "ops.h"

namespace rwkv {

namespace {

constexpr int kLpThreads = 256;

struct LogprobArgs {
  const void* logits;
  int64_t ld;
  const int* tokens;
  float* logprob;
  float* entropy;
  int* rank;
  int* top_ids;
  float* top_logprobs;
  int V, top_n;
};

template <typename T>
__global__ __launch_bounds__(kLpThreads) void token_logprobs_kernel(LogprobArgs a) {
  __shared__ float red[4][kLpThreads / 64];
  __shared__ int idx[kLpThreads / 64];
  const T* z = static_cast<const T*>(a.logits) + blockIdx.x * a.ld;
  const int V = a.V;
  auto at = [&](int i) { return static_cast<float>(z[i]); };
  auto block_max = [&](float v, int slot) {
    v = wave_reduce_dpp(v, [](float x, float y) { return fmaxf(x, y); });
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[slot][threadIdx.x >> 6] = v;
    __syncthreads();
    float r = red[slot][0];
#pragma unroll
    for (int i = 1; i < kLpThreads / 64; ++i) r = fmaxf(r, red[slot][i]);
    return r;
  };
  float m = -INFINITY;
  for (int i = threadIdx.x; i < V; i += kLpThreads) m = fmaxf(m, at(i));
  m = block_max(m, 0);
  const int t = a.tokens ? a.tokens[blockIdx.x] : -1;
  const float zt = t >= 0 && t < V ? at(t) : 0.0f;
  float s = 0.0f, u = 0.0f, ahead = 0.0f;
  for (int i = threadIdx.x; i < V; i += kLpThreads) {
    const float x = at(i);
    float d = x - m;
    if (d < -200.0f) d = -200.0f;  // e^-200 is 0 in fp32, and 0 times an infinity is none
    if (x == -INFINITY) d = -200.0f;
    const float e = __expf(d);
    s += e;
    u = fmaf(d, e, u);
    if (x > zt || (x == zt && i < t)) ahead += 1.0f;
  }
  s = block_sum<kLpThreads / 64>(s, red[1]);
  u = block_sum<kLpThreads / 64>(u, red[2]);
  ahead = block_sum<kLpThreads / 64>(ahead, red[3]);
  const bool nothing = m == -INFINITY && s == 0.0f;
  const float log_s = logf(s);
  if (threadIdx.x == 0) {
    if (a.logprob) a.logprob[blockIdx.x] = t < 0 ? 0.0f : t >= V ? __builtin_nanf("") : nothing ? -INFINITY : zt - m - log_s;
    if (a.entropy) a.entropy[blockIdx.x] = nothing ? 0.0f : log_s - u / s;
    if (a.rank) a.rank[blockIdx.x] = t < 0 || t >= V || zt != zt ? -1 : static_cast<int>(ahead);
  }
  // the alternatives one after the other: the first entry behind the one before
  float last = INFINITY;
  int last_i = -1;
  for (int k = 0; k < a.top_n; ++k) {
    float best = -INFINITY;
    int bi = V;
    for (int i = threadIdx.x; i < V; i += kLpThreads) {
      const float x = at(i);
      if ((x < last || (x == last && i > last_i)) && x > best) {
        best = x;
        bi = i;
      }
    }
    const float top = block_max(best, 0);
    bi = best == top ? bi : V;
    bi = wave_reduce_dpp(bi, [](int x, int y) { return min(x, y); });
    __syncthreads();
    if ((threadIdx.x & 63) == 0) idx[threadIdx.x >> 6] = bi;
    __syncthreads();
    for (int i = 0; i < kLpThreads / 64; ++i) bi = min(bi, idx[i]);
    if (threadIdx.x == 0) {
      const int64_t o = static_cast<int64_t>(blockIdx.x) * a.top_n + k;
      a.top_ids[o] = bi < V ? bi : -1;
      a.top_logprobs[o] = bi < V ? top - m - log_s : -INFINITY;
    }
    last = top;
    last_i = bi;
  }
}

}  // namespace

size_t token_logprobs_workspace_bytes(int rows, int V, int top_n) { return 0; }

int token_logprobs_launch(hipStream_t st, int rows, int V, int io, const void* logits, int64_t ld, const TokenLogprobs& out, void* workspace) {
  LogprobArgs a = {logits, ld, out.tokens, out.logprob, out.entropy, out.rank, out.top_ids, out.top_logprobs, V, out.top_n};
  if (io == RWKV_IO_F16) hipLaunchKernelGGL(token_logprobs_kernel<half_t>, dim3(rows), dim3(kLpThreads), 0, st, a);
  else hipLaunchKernelGGL(token_logprobs_kernel<float>, dim3(rows), dim3(kLpThreads), 0, st, a);
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
