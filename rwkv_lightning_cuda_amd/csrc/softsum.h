// What the two files of the log probabilities share: the running sums of a softmax and its entropy, and the results they give.
#pragma once

#include "ops.h"

namespace rwkv {

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLowest = -3.402823466e38f;
constexpr float kGone = -200.0f;  // e^-200 is 0 in fp32; a difference that is multiplied by it must not be infinite

// m = max z, S = sum e^(z - m), U = sum (z - m) e^(z - m) of the entries seen so far.  m starts at the lowest finite value, not at
// -infinity: differences with it are no NaN, and S stays 0 as long as every entry is -infinity.  A NaN or +infinity among the entries
// makes S a NaN that stays.
struct SoftSum {
  float m = kLowest, s = 0.0f, u = 0.0f;
  __device__ __forceinline__ void raise(float to) {
    const float t = fmaxf(m - to, kGone);
    const float f = __builtin_amdgcn_exp2f(t * kLog2e);
    u = f * fmaf(t, s, u);
    s *= f;
    m = to;
  }
  // first, o_first: where each has its largest entry; the lower one where they are equal
  __device__ __forceinline__ void merge(SoftSum o, int& first, int o_first) {
    first = o.m > m ? o_first : (o.m == m ? min(first, o_first) : first);
    const float to = fmaxf(m, o.m);
    raise(to);
    o.raise(to);
    s += o.s;
    u += o.u;
  }
};

// by value, as as_half2: a bit cast of a vector's element reads element 0
__device__ __forceinline__ int as_int(float v) { return __builtin_bit_cast(int, v); }

// whether entry i of value v is ahead of entry k of value w
__device__ __forceinline__ bool ahead_of(float v, int i, float w, int k) { return v > w || (v == w && i < k); }

// log probability and entropy of a row: ln S - U / S is a sum of two terms that are not negative, nothing cancels.  token_logit is
// that of the row's token, read only where it is an entry
__device__ __forceinline__ void write_logprobs(const SoftSum& a, const TokenLogprobs& out, int64_t row, int V, const float* token_logit) {
  const bool nothing = a.s == 0.0f;
  const float log_s = logf(a.s);
  if (out.logprob) {
    const int t = out.tokens[row];
    out.logprob[row] = t < 0 ? 0.0f : t >= V ? __builtin_nanf("") : nothing ? -INFINITY : *token_logit - a.m - log_s;
  }
  if (out.entropy) out.entropy[row] = nothing ? 0.0f : log_s - a.u / a.s;
}

}  // namespace rwkv
