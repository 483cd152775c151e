// The vocabulary's product with the log probabilities of its logits: z[M,N] = x[M,K] . W[N,K]^T in fp32 (not rounded to fp16 as the
// logits of a forward pass are), then what logprobs.hip makes of the rows.  x fp16 with fp16 or int8 weights, or int8 codes with a
// scale per row and int8 weights (products in whole numbers, exact in 32 bits up to K = 133152: 127 * 127 K < 2^31).
// Reference: the head product alone (src/rwkv7_fast_v4.cu:1325-1341).
#include "gemm_stream.h"

namespace rwkv {

namespace {

typedef int int4v_t __attribute__((ext_vector_type(4)));
typedef int int16v_t __attribute__((ext_vector_type(16)));

enum { kF16F16 = 0, kF16W8 = 1, kI8W8 = 2 };

struct HeadArgs {
  const void* x;         // [M,K] fp16 or int8
  const float* x_scale;  // int8: [M]
  const uint4_t* wp;     // packed
  const half_t* scale;   // int8 weights: [N]
  float* logits;         // [M,N]
  int M, N, K;
};

// A wavefront per 32 rows and 32 columns.  The packed order gives a lane (j, h) the codes k = 32 g + 16 h .. + 15 of column j of its
// band; it takes the same k of row j of x.
template <int TYPES>
__global__ __launch_bounds__(256) void head_logits_kernel(HeadArgs g) {
  const int lane = threadIdx.x & 63, j = lane & 31, h = lane >> 5;
  const int band = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (band * 32 >= g.N) return;
  const int row = blockIdx.y * 32 + j;
  const int row_read = row < g.M ? row : g.M - 1;
  const int groups = g.K / 32;
  constexpr int kPieces = TYPES == kF16F16 ? 2 : 1;
  const uint4_t* w = g.wp + static_cast<int64_t>(band) * groups * kPieces * 64 + lane;
  const char* x = static_cast<const char*>(g.x) + static_cast<int64_t>(row_read) * g.K * (TYPES == kI8W8 ? 1 : 2) + h * (TYPES == kI8W8 ? 16 : 32);
  float z[16];
  if constexpr (TYPES == kI8W8) {
    int16v_t acc;
#pragma unroll
    for (int v = 0; v < 16; ++v) acc[v] = 0;
    for (int c = 0; c < groups; ++c)
      acc = __builtin_amdgcn_mfma_i32_32x32x32_i8(__builtin_bit_cast(int4v_t, w[c * 64]), *reinterpret_cast<const int4v_t*>(x + c * 32), acc, 0, 0, 0);
#pragma unroll
    for (int v = 0; v < 16; ++v) z[v] = static_cast<float>(acc[v]);
  } else {
    float16_t acc;
#pragma unroll
    for (int v = 0; v < 16; ++v) acc[v] = 0.0f;
    for (int c = 0; c < groups; ++c) {
      half8_t b0, b1;
      if constexpr (TYPES == kF16F16) {
        b0 = __builtin_bit_cast(half8_t, w[c * 128]);
        b1 = __builtin_bit_cast(half8_t, w[c * 128 + 64]);
      } else {
        const uint4_t p = w[c * 64];
        b0 = expand_w8(p[0], p[1]);
        b1 = expand_w8(p[2], p[3]);
      }
      const half8_t* xs = reinterpret_cast<const half8_t*>(x + c * 64);
      acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(b0, xs[0], acc, 0, 0, 0);
      acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(b1, xs[1], acc, 0, 0, 0);
    }
#pragma unroll
    for (int v = 0; v < 16; ++v) z[v] = acc[v];
  }
  if (row >= g.M) return;
  const float xs = TYPES == kI8W8 ? g.x_scale[row] : 1.0f;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int col = band * 32 + 8 * q + 4 * h;
    float4_t out;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      out[i] = z[4 * q + i];
      if constexpr (TYPES != kF16F16) out[i] *= h2f(g.scale[col + i]);
      if constexpr (TYPES == kI8W8) out[i] *= xs;
    }
    *reinterpret_cast<float4_t*>(g.logits + static_cast<int64_t>(row) * g.N + col) = out;
  }
}

constexpr int kBlockRows = 256;  // rows whose logits exist at a time

int rows_at_a_time(int M) { return M < kBlockRows ? M : kBlockRows; }
size_t align16(size_t n) { return (n + 15) / 16 * 16; }

}  // namespace

size_t linear_logprobs_workspace_bytes(int fmt, bool x_int8, int M, int N, int K, int top_n) {
  const int rows = rows_at_a_time(M);
  return align16(static_cast<size_t>(rows) * N * 4) + token_logprobs_workspace_bytes(rows, N, top_n);
}

int linear_logprobs_launch(hipStream_t st, int fmt, int M, int N, int K, const void* x, const float* x_scale, const void* packed,
                           const half_t* scale, const TokenLogprobs& out, void* workspace) {
  const int step = rows_at_a_time(M);
  float* logits = static_cast<float*>(workspace);
  unsigned char* rest = static_cast<unsigned char*>(workspace) + align16(static_cast<size_t>(step) * N * 4);
  for (int m = 0; m < M; m += step) {
    const int rows = M - m < step ? M - m : step;
    const int64_t off = static_cast<int64_t>(m) * K;
    HeadArgs g = {static_cast<const char*>(x) + off * (x_scale ? 1 : 2), x_scale ? x_scale + m : nullptr, static_cast<const uint4_t*>(packed),
                  scale, logits, rows, N, K};
    const dim3 grid(ceil_div(N, 128), ceil_div(rows, 32));
    if (x_scale) hipLaunchKernelGGL(head_logits_kernel<kI8W8>, grid, dim3(256), 0, st, g);
    else if (fmt == RWKV_FMT_W8) hipLaunchKernelGGL(head_logits_kernel<kF16W8>, grid, dim3(256), 0, st, g);
    else hipLaunchKernelGGL(head_logits_kernel<kF16F16>, grid, dim3(256), 0, st, g);
    RWKV_LAUNCH_CHECK();
    const int rc = token_logprobs_launch(st, rows, N, RWKV_IO_F32, logits, N, out.from_row(m), rest);
    if (rc != RWKV_OK) return rc;
  }
  return RWKV_OK;
}

namespace {

int check_shape(const char* who, int fmt, bool x_int8, int M, int N, int K) {
  RWKV_REQUIRE(fmt == RWKV_FMT_F16 || fmt == RWKV_FMT_W8, "%s: weights are fp16 or int8, got format %d", who, fmt);
  RWKV_REQUIRE(!x_int8 || fmt == RWKV_FMT_W8, "%s: int8 x needs int8 weights", who);
  RWKV_REQUIRE(M > 0, "%s: M must be positive, got %d", who, M);
  RWKV_REQUIRE(linear_packed_supported(fmt, M, N, K), "%s: unsupported shape N=%d K=%d (multiples of 32 and 256)", who, N, K);
  RWKV_REQUIRE(N <= kMaxLogprobVocab && K <= 16384, "%s: N up to %d and K up to 16384, got %d and %d", who, kMaxLogprobVocab, N, K);
  return RWKV_OK;
}

}  // namespace

}  // namespace rwkv

using namespace rwkv;

extern "C" {

int rwkv_hip_linear_logprobs_workspace(int fmt, int x_int8, int M, int N, int K, int top_n, size_t* bytes) {
  RWKV_REQUIRE(bytes, "linear_logprobs_workspace: NULL result");
  const int rc = check_shape("linear_logprobs_workspace", fmt, x_int8 != 0, M, N, K);
  if (rc != RWKV_OK) return rc;
  RWKV_REQUIRE(top_n >= 0 && top_n <= kMaxAlternatives, "linear_logprobs_workspace: top_n must lie in 0 .. %d, got %d", kMaxAlternatives, top_n);
  *bytes = linear_logprobs_workspace_bytes(fmt, x_int8 != 0, M, N, K, top_n);
  return RWKV_OK;
}

int rwkv_hip_linear_logprobs(rwkv_stream_t s, int fmt, int M, int N, int K, const void* x, const void* x_scale, const void* packed,
                             const void* scale, const void* tokens, int top_n, void* logprob, void* entropy, void* top_ids,
                             void* top_logprobs, void* workspace, size_t workspace_bytes) {
  int rc = check_shape("linear_logprobs", fmt, x_scale != nullptr, M, N, K);
  if (rc != RWKV_OK) return rc;
  RWKV_REQUIRE(x && packed && (fmt == RWKV_FMT_F16 || scale), "linear_logprobs: NULL tensor");
  RWKV_REQUIRE(((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(packed)) & 15) == 0 &&
                   (reinterpret_cast<uintptr_t>(scale) & 7) == 0 && (reinterpret_cast<uintptr_t>(x_scale) & 3) == 0,
               "linear_logprobs: x and packed must be aligned to 16 bytes, scale to 8, x_scale to 4");
  const TokenLogprobs out = {static_cast<const int*>(tokens), top_n, static_cast<float*>(logprob), static_cast<float*>(entropy),
                             nullptr, static_cast<int*>(top_ids), static_cast<float*>(top_logprobs)};
  rc = check_token_logprobs("linear_logprobs", out);
  if (rc != RWKV_OK) return rc;
  const size_t need = linear_logprobs_workspace_bytes(fmt, x_scale != nullptr, M, N, K, top_n);
  RWKV_REQUIRE(workspace && workspace_bytes >= need && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0,
               "linear_logprobs: workspace of %zu bytes (aligned to 16) needed, got %zu", need, workspace_bytes);
  return linear_logprobs_launch(as_stream(s), fmt, M, N, K, x, static_cast<const float*>(x_scale), packed, static_cast<const half_t*>(scale), out,
                                workspace);
}

}  // extern "C"
