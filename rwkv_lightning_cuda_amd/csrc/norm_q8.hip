// Residual addition, LayerNorm or root-mean-square norm, and an 8-bit output with a scale per row: the input of a product whose
// weights are int8 codes as well.  No counterpart in the reference, whose norms write fp16 (cuda/rwkv7_v3a_ops.cu:1272-1351).
//
//   s = x + res (fp32);  x_out = f16(s)
//   c = s - mean(s) (layer) or s (rms);  y = c / sqrt(mean(c^2) + eps) * w + b, unrounded
//   scale = max|y| / 127;  q = rint(y / scale), ties to even;  scale = 0 and q = 0 where max|y| = 0
//   a row whose y is not finite somewhere: scale = NaN and q = 0, so that whatever reads it is NaN too
//
// Bound by memory: 7 bytes a value, 2048 rows of 4096 (58.7 MB) 12.5 us = 4.7 TB/s, where a large copy moves 4.9; few rows by the launch
// (one row of 768 2.4 us) and three block-wide reductions behind one trip to memory.
//
// y stays in fp32 from the sum to the code: an fp16 y in between would add half a step of 2^-11 of the value, an eighth of the
// code's own rounding at the largest values.
#include "ops.h"

namespace rwkv {

namespace {

struct NormQ8Args {
  const half_t* x;
  const half_t* res;  // may be NULL
  const half_t* w;
  const half_t* b;    // may be NULL
  half_t* x_out;      // may be NULL
  int8_t* q;
  float* scale;
  int rows, C;
  float eps;
};

// the larger one, NaN if either is
__device__ __forceinline__ float max_or_nan(float a, float b) { return (b > a || b != b) ? b : a; }

// One block per row, eight values per thread.
template <bool RMS, int NT>
__global__ __launch_bounds__(NT) void norm_q8_kernel(NormQ8Args a) {
  __shared__ float red[3][NT / 64];
  const int c = threadIdx.x * 8;
  const bool live = c < a.C;
  const int64_t o = static_cast<int64_t>(blockIdx.x) * a.C + (live ? c : 0);
  const half8_t xv = *reinterpret_cast<const half8_t*>(a.x + o);
  half8_t rv = {}, bv = {};
  const half8_t wv = *reinterpret_cast<const half8_t*>(a.w + (live ? c : 0));
  if (a.res) rv = *reinterpret_cast<const half8_t*>(a.res + o);
  if (a.b) bv = *reinterpret_cast<const half8_t*>(a.b + (live ? c : 0));
  float v[8];
  float sum = 0.0f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    v[e] = live ? h2f(xv[e]) + h2f(rv[e]) : 0.0f;
    sum += v[e];
  }
  if (a.x_out && live) {
    half8_t xo;
#pragma unroll
    for (int e = 0; e < 8; ++e) xo[e] = f2h(v[e]);
    *reinterpret_cast<half8_t*>(a.x_out + o) = xo;
  }
  if constexpr (!RMS) {
    const float mean = block_sum<NT / 64>(sum, red[0]) / static_cast<float>(a.C);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = live ? v[e] - mean : 0.0f;
  }
  float sq = 0.0f;
#pragma unroll
  for (int e = 0; e < 8; ++e) sq = fmaf(v[e], v[e], sq);
  const float rstd = rsqrtf(block_sum<NT / 64>(sq, red[1]) / static_cast<float>(a.C) + a.eps);
  float amax = 0.0f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    v[e] = fmaf(v[e] * rstd, h2f(wv[e]), h2f(bv[e]));
    if (live) amax = max_or_nan(amax, fabsf(v[e]));
  }
  amax = wave_reduce_dpp(amax, max_or_nan);
  if constexpr (NT > 64) {
    if ((threadIdx.x & 63) == 0) red[2][threadIdx.x >> 6] = amax;
    __syncthreads();
    amax = red[2][0];
#pragma unroll
    for (int i = 1; i < NT / 64; ++i) amax = max_or_nan(amax, red[2][i]);
  }
  const bool fine = amax < INFINITY;  // false for NaN
  const float inv = fine && amax > 0.0f ? 127.0f / amax : 0.0f;
  if (threadIdx.x == 0) a.scale[blockIdx.x] = fine ? amax / 127.0f : __builtin_nanf("");
  if (!live) return;
  uint2_t packed = {0, 0};
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int code = fine ? static_cast<int>(rintf(v[e] * inv)) : 0;
    packed[e >> 2] |= (static_cast<uint32_t>(code) & 0xffu) << (8 * (e & 3));
  }
  *reinterpret_cast<uint2_t*>(a.q + o) = packed;
}

template <bool RMS>
int launch(hipStream_t st, const NormQ8Args& a) {
  const dim3 grid(a.rows);
  if (a.C <= 512) hipLaunchKernelGGL((norm_q8_kernel<RMS, 64>), grid, dim3(64), 0, st, a);
  else if (a.C <= 2048) hipLaunchKernelGGL((norm_q8_kernel<RMS, 256>), grid, dim3(256), 0, st, a);
  else if (a.C <= 4096) hipLaunchKernelGGL((norm_q8_kernel<RMS, 512>), grid, dim3(512), 0, st, a);
  else hipLaunchKernelGGL((norm_q8_kernel<RMS, 1024>), grid, dim3(1024), 0, st, a);
  RWKV_LAUNCH_CHECK();
  return RWKV_OK;
}

}  // namespace

}  // namespace rwkv

using namespace rwkv;

extern "C" int rwkv_hip_add_norm_q8(rwkv_stream_t s, int rows, int C, int norm, const void* x, const void* res, const void* w,
                                    const void* b, float eps, void* x_out, void* q, void* scale) {
  RWKV_REQUIRE(norm == RWKV_NORM_LAYER || norm == RWKV_NORM_RMS, "add_norm_q8: unknown norm %d", norm);
  RWKV_REQUIRE(rows > 0, "add_norm_q8: rows must be positive, got %d", rows);
  RWKV_REQUIRE(C > 0 && C % 8 == 0 && C <= 8192, "add_norm_q8: C must be a multiple of 8 up to 8192, got %d", C);
  RWKV_REQUIRE(x && w && q && scale, "add_norm_q8: NULL tensor");
  RWKV_REQUIRE(eps >= 0.0f, "add_norm_q8: eps must not be negative");
  for (const void* p : {x, res, w, b, static_cast<const void*>(x_out)})
    RWKV_REQUIRE((reinterpret_cast<uintptr_t>(p) & 15) == 0, "add_norm_q8: fp16 tensors must be aligned to 16 bytes");
  RWKV_REQUIRE((reinterpret_cast<uintptr_t>(q) & 7) == 0 && (reinterpret_cast<uintptr_t>(scale) & 3) == 0,
               "add_norm_q8: q must be aligned to 8 bytes, scale to 4");
  NormQ8Args a = {static_cast<const half_t*>(x), static_cast<const half_t*>(res), static_cast<const half_t*>(w),
                  static_cast<const half_t*>(b), static_cast<half_t*>(x_out), static_cast<int8_t*>(q), static_cast<float*>(scale),
                  rows, C, eps};
  return norm == RWKV_NORM_RMS ? launch<true>(as_stream(s), a) : launch<false>(as_stream(s), a);
}
