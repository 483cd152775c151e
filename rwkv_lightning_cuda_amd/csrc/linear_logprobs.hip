// The vocabulary's product with the log probabilities of its logits: z[M,N] = x[M,K] . W[N,K]^T in fp32 (not rounded to fp16 as the
// logits of a forward pass are), then what logprobs.hip makes of the rows.  x fp16 with fp16 or int8 weights, or int8 codes with a
// scale per row and int8 weights (products in whole numbers, exact in 32 bits up to K = 133152: 127 * 127 K < 2^31).
// Reference: the head product alone (src/rwkv7_fast_v4.cu:1325-1341).
#include <algorithm>

#include "gemm_tile.h"
#include "softsum.h"

namespace rwkv {

namespace {

enum { kF16F16 = 0, kF16W8 = 1, kI8W8 = 2 };
template <int TYPES>
struct Types {
  static constexpr int kTile = TYPES == kF16F16 ? RWKV_FMT_F16 : TYPES == kF16W8 ? RWKV_FMT_W8 : kTileI8;
  static constexpr int kXBytes = TYPES == kI8W8 ? 1 : 2;       // of a value of x
  static constexpr int kPieces = TYPES == kF16F16 ? 2 : 1;     // 1 KiB weight pieces of 32 columns and 32 k
  static constexpr int kBandBytes = kPieces * 32;              // of 32 columns and one k
};

struct HeadArgs {
  const char* x;         // [M,K] fp16 or int8
  const float* x_scale;  // int8: [M]
  const char* wp;        // packed
  const half_t* scale;   // int8 weights: [N]
  int M, N, K;
  float* logits;         // [M,N]
  // sums of the tiles instead of logits
  const int* tokens;     // may be NULL
  float4_t* part;        // [blocks of 256 columns][M]: m, S, U and the first column of value m
  float* token_logit;    // [M], written where the token is a column
  bool want_first;
  int row_tiles, col_blocks;
};

__device__ __forceinline__ int other_half(int v) { return lane_xor_dpp<32>(v); }
__device__ __forceinline__ float other_half(float v) { return __builtin_bit_cast(float, lane_xor_dpp<32>(__builtin_bit_cast(int, v))); }

// ---- few rows: the weights are streamed once, which is what bounds it ------------------------------------------------
// A wavefront takes whole bands of 32 columns, one after the other in memory, 8 KiB of them requested ahead of the 8 KiB that it
// multiplies.  x lies in LDS in the order in which the matrix core's lanes read it - lane (j, h) the 16 bytes of row j & (R - 1), k =
// 32 g + 16 h (int8) or + 8 i (fp16) - R = the rows rounded up to a power of two.
constexpr int kFewThreads = 512;
constexpr int kFewLds = 128 * 1024;
constexpr int kFewRows = 32;

int few_rows(int M) {
  int r = 1;
  while (r < M) r *= 2;
  return r;
}
bool takes_few(int M, int K, int x_bytes) { return M <= kFewRows && static_cast<int64_t>(few_rows(M)) * K * x_bytes <= kFewLds; }

template <int TYPES>
__global__ __launch_bounds__(kFewThreads) void head_few_kernel(HeadArgs g, int log_rows, int bands_per_wave) {
  typedef Types<TYPES> T;
  extern __shared__ __align__(16) unsigned char x_lds[];
  constexpr int kWaves = kFewThreads / 64;
  constexpr int kChunk = 8;                 // pieces
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int lane = threadIdx.x & 63, j = lane & 31, h = lane >> 5;
  const int bands = g.N / 32;
  const int band0 = (blockIdx.x * kWaves + wave) * bands_per_wave;
  const int band1 = min(band0 + bands_per_wave, bands);
  const int band_pieces = g.K / 32 * T::kPieces;
  const int chunks = (band1 - band0) * (band_pieces / kChunk);
  const uint4_t* w = reinterpret_cast<const uint4_t*>(g.wp) + static_cast<int64_t>(band0) * band_pieces * 64 + lane;
  uint4_t ahead[kChunk];
  auto request = [&]() {
#pragma unroll
    for (int p = 0; p < kChunk; ++p) ahead[p] = w[p * 64];
    w += kChunk * 64;
  };
  if (chunks > 0) request();
  // x: 16-byte piece n of row r holds k = n * 16 / kXBytes ..; its place is [n / 2 (int8) or n / 4 and n % 2][h][row]
  {
    const int row_pieces = g.K * T::kXBytes / 16;
    const int R = 1 << log_rows;
    for (int i = threadIdx.x; i < row_pieces << log_rows; i += kFewThreads) {
      const int r = i / row_pieces, n = i - r * row_pieces;
      const int row = min(r, g.M - 1);
      const int place = TYPES == kI8W8 ? n : (n & ~3) | ((n & 1) << 1) | ((n >> 1) & 1);
      *reinterpret_cast<uint4_t*>(x_lds + (static_cast<int64_t>(place) * R + r) * 16) =
          *reinterpret_cast<const uint4_t*>(g.x + static_cast<int64_t>(row) * g.K * T::kXBytes + n * 16);
    }
  }
  __syncthreads();
  const int R = 1 << log_rows;
  const uint32_t x_lane = ((h << log_rows) + (j & (R - 1))) * 16;
  const uint32_t x_step = 2u * 16u << log_rows;  // from one product's fragment to the next
  const float xs = TYPES == kI8W8 ? g.x_scale[min(j, g.M - 1)] : 1.0f;
  typedef typename WideTile<T::kTile, 2>::acc_t acc_t;
  int left = chunks;
  for (int band = band0; band < band1; ++band) {
    acc_t acc;
#pragma unroll
    for (int v = 0; v < 16; ++v) acc[v] = 0;
    uint32_t at = x_lane;
    for (int c = 0; c < band_pieces / kChunk; ++c) {
      uint4_t now[kChunk];
#pragma unroll
      for (int p = 0; p < kChunk; ++p) now[p] = ahead[p];
      if (--left > 0) request();
#pragma unroll
      for (int p = 0; p < kChunk; ++p) {
        if constexpr (TYPES == kI8W8) {
          acc = __builtin_amdgcn_mfma_i32_32x32x32_i8(__builtin_bit_cast(int4v_t, now[p]), *reinterpret_cast<const int4v_t*>(x_lds + at), acc, 0, 0, 0);
          at += x_step;
        } else if constexpr (TYPES == kF16F16) {
          acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8_t, now[p]), *reinterpret_cast<const half8_t*>(x_lds + at), acc, 0, 0, 0);
          at += x_step;
        } else {
          acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(expand_w8(now[p][0], now[p][1]), *reinterpret_cast<const half8_t*>(x_lds + at), acc, 0, 0, 0);
          at += x_step;
          acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(expand_w8(now[p][2], now[p][3]), *reinterpret_cast<const half8_t*>(x_lds + at), acc, 0, 0, 0);
          at += x_step;
        }
      }
    }
    if (j < g.M) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int col = band * 32 + 8 * q + 4 * h;
        float4_t out;
#pragma unroll
        for (int i = 0; i < 4; ++i) out[i] = static_cast<float>(acc[4 * q + i]);
        if constexpr (TYPES != kF16F16) {
          const half4_t sc = *reinterpret_cast<const half4_t*>(g.scale + col);
#pragma unroll
          for (int i = 0; i < 4; ++i) out[i] = mul_f32(out[i], h2f(sc[i]));
        }
        if constexpr (TYPES == kI8W8) {
#pragma unroll
          for (int i = 0; i < 4; ++i) out[i] = mul_f32(out[i], xs);
        }
        *reinterpret_cast<float4_t*>(g.logits + static_cast<int64_t>(j) * g.N + col) = out;
      }
    }
  }
}

// ---- many rows: the tiles of the packed product -----------------------------------------------------------------------
// SUMS: a tile leaves m, S and U of its 256 columns for every row (16 bytes for 1 KiB of logits), otherwise the logits.
// A lane has 32 columns of a row in registers: they are reduced there, with the other half's 32 by a swap of rows, with the other
// three wavefronts' 64 each through LDS.
template <int TYPES, int MT, bool SUMS>
__global__ __launch_bounds__(64 * kTileWaves, 2) void head_tile_kernel(HeadArgs g) {
  typedef Types<TYPES> T;
  typedef WideTile<T::kTile, MT> W;
  __shared__ __align__(1024) unsigned char lds[W::kStages * W::kStageBytes];
  const int id = blockIdx.x;
  const int row_tile = (id >> 3) % g.row_tiles;
  const int col_block = (id / (8 * g.row_tiles)) * 8 + (id & 7);
  if (col_block >= g.col_blocks) return;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int lane = threadIdx.x & 63, j = lane & 31, h = lane >> 5;
  const int wm = wave & 1, wn = wave >> 1;
  const int m0 = row_tile * W::BM;
  const int band = min(col_block * 8 + wave, g.N / 32 - 1);  // past the last band: repeat it
  typename W::acc_t acc[2][MT];
  tile_products<T::kTile, MT>(g.x + static_cast<int64_t>(m0) * g.K * T::kXBytes, static_cast<uint32_t>(g.K) * T::kXBytes, g.M - m0,
                              g.wp + static_cast<int64_t>(band) * g.K * T::kBandBytes, g.K / W::kK, lds, acc);

  const int col0 = col_block * kTileCols + wn * 64;
  half4_t sc[2][4];
#pragma unroll
  for (int nb = 0; nb < 2; ++nb)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      sc[nb][q] = half4_t{1, 1, 1, 1};
      if (TYPES != kF16F16) sc[nb][q] = *reinterpret_cast<const half4_t*>(g.scale + min(col0 + nb * 32, g.N - 32) + 8 * q + 4 * h);
    }
  float4_t* merge = reinterpret_cast<float4_t*>(lds);  // [4][BM]
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    const int r = (wm * MT + mt) * 32 + j;
    const int row = m0 + r;
    const bool live = row < g.M;
    const float xs = TYPES == kI8W8 ? g.x_scale[live ? row : g.M - 1] : 1.0f;
    float z[2][16];
#pragma unroll
    for (int nb = 0; nb < 2; ++nb)
#pragma unroll
      for (int v = 0; v < 16; ++v) {
        z[nb][v] = static_cast<float>(acc[nb][mt][v]);
        if (TYPES != kF16F16) z[nb][v] = mul_f32(z[nb][v], h2f(sc[nb][v >> 2][v & 3]));
      }
    if constexpr (!SUMS) {
      if (!live) continue;
#pragma unroll
      for (int nb = 0; nb < 2; ++nb)
        if (col0 + nb * 32 < g.N) {
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            float4_t out = {z[nb][4 * q], z[nb][4 * q + 1], z[nb][4 * q + 2], z[nb][4 * q + 3]};
            if (TYPES == kI8W8) {
#pragma unroll
              for (int i = 0; i < 4; ++i) out[i] = mul_f32(out[i], xs);
            }
            *reinterpret_cast<float4_t*>(g.logits + static_cast<int64_t>(row) * g.N + col0 + nb * 32 + 8 * q + 4 * h) = out;
          }
        }
    } else {
      // the largest column, and the first of its value (in units of x_scale, as everything up to the exponent)
      float m = kLowest;
      int first = 0;
#pragma unroll
      for (int nb = 0; nb < 2; ++nb)
        if (col0 + nb * 32 < g.N) {
#pragma unroll
          for (int v = 0; v < 16; ++v) m = fmaxf(m, z[nb][v]);
        }
      if (g.want_first) {
#pragma unroll
        for (int nb = 1; nb >= 0; --nb)
          if (col0 + nb * 32 < g.N) {
#pragma unroll
            for (int v = 15; v >= 0; --v)
              if (z[nb][v] == m) first = nb * 32 + 8 * (v >> 2) + (v & 3);
          }
        first += col0 + 4 * h;
      }
      const float to_log2 = xs * kLog2e;
      float s = 0.0f, u = 0.0f;
#pragma unroll
      for (int nb = 0; nb < 2; ++nb)
        if (col0 + nb * 32 < g.N) {
#pragma unroll
          for (int v = 0; v < 16; ++v) {
            const float d = z[nb][v] - m;
            const float p = __builtin_amdgcn_exp2f(d * to_log2);
            s += p;
            u = fmaf(fmaxf(d, kLowest), p, u);
          }
        }
      const int t = g.tokens && live ? g.tokens[row] - col0 : -1;
      if (t >= 0 && t < 64 && ((t >> 2) & 1) == h && col0 + t < g.N) {
        float zt = 0.0f;
#pragma unroll
        for (int nb = 0; nb < 2; ++nb)
#pragma unroll
          for (int v = 0; v < 16; ++v)
            if (t - 4 * h == nb * 32 + 8 * (v >> 2) + (v & 3)) zt = z[nb][v];
        g.token_logit[row] = mul_f32(zt, xs);
      }
      // both halves in one
      SoftSum a = {m * xs, s, u * xs};
      if (m == kLowest) a = {kLowest, s, 0.0f};
      a.merge(SoftSum{other_half(a.m), other_half(a.s), other_half(a.u)}, first, other_half(first));
      if (h == 0) merge[wn * W::BM + r] = float4_t{a.m, a.s, a.u, __builtin_bit_cast(float, first)};
    }
  }
  if constexpr (SUMS) {
    __syncthreads();
    const int r = threadIdx.x;
    if (r < W::BM && m0 + r < g.M) {
      const float4_t p = merge[r];
      SoftSum a = {p[0], p[1], p[2]};
      int first = as_int(p[3]);
#pragma unroll
      for (int i = 1; i < 4; ++i) {
        const float4_t o = merge[i * W::BM + r];
        a.merge(SoftSum{o[0], o[1], o[2]}, first, as_int(o[3]));
      }
      g.part[static_cast<int64_t>(col_block) * g.M + m0 + r] = float4_t{a.m, a.s, a.u, __builtin_bit_cast(float, first)};
    }
  }
}

// 16 rows per block, 16 threads per row over the blocks of columns
__global__ __launch_bounds__(256) void head_join_kernel(HeadArgs g, TokenLogprobs out) {
  __shared__ float4_t parts[16][17];
  const int r = threadIdx.x & 15, i = threadIdx.x >> 4;
  const int row = blockIdx.x * 16 + r;
  SoftSum a;
  int first = 0;
  if (row < g.M) {
    for (int c = i; c < g.col_blocks; c += 16) {
      const float4_t p = g.part[static_cast<int64_t>(c) * g.M + row];
      a.merge(SoftSum{p[0], p[1], p[2]}, first, as_int(p[3]));
    }
  }
  parts[r][i] = float4_t{a.m, a.s, a.u, __builtin_bit_cast(float, first)};
  __syncthreads();
  if (threadIdx.x >= 16 || row >= g.M) return;
  for (int k = 1; k < 16; ++k) {
    const float4_t p = parts[r][k];
    a.merge(SoftSum{p[0], p[1], p[2]}, first, as_int(p[3]));
  }
  write_logprobs(a, out, row, g.N, g.token_logit + row);
  if (out.top_n == 1) {
    const bool there = a.m > kLowest;
    out.top_ids[row] = there ? first : -1;
    out.top_logprobs[row] = there ? -logf(a.s) : -INFINITY;
  }
}

// ---- what a call takes ------------------------------------------------------------------------------------------------
enum Way { kFew, kLogits, kSums };
struct Plan {
  Way way;
  int rows;      // at a time
  size_t logits, part, token_logit;  // bytes, of 256 each
  size_t rest;
  size_t bytes() const { return logits + part + token_logit + rest; }
};

constexpr int kLogitRows = 256;  // rows whose logits exist at a time
constexpr int kSumRows = 8192;   // rows whose tiles' sums do

Plan plan_of(bool x_int8, int M, int N, int K, int top_n) {
  Plan p = {};
  p.way = takes_few(M, K, x_int8 ? 1 : 2) ? kFew : top_n > 1 ? kLogits : kSums;
  p.rows = p.way == kFew ? M : std::min(M, p.way == kSums ? kSumRows : kLogitRows);
  const auto align = [](size_t n) { return (n + 255) / 256 * 256; };
  if (p.way == kSums) {
    p.part = align(static_cast<size_t>(ceil_div(N, kTileCols)) * p.rows * sizeof(float4_t));
    p.token_logit = align(static_cast<size_t>(p.rows) * 4);
  } else {
    p.logits = align(static_cast<size_t>(p.rows) * N * 4);
    p.rest = token_logprobs_workspace_bytes(p.rows, N, top_n);
  }
  return p;
}

template <int TYPES>
int launch_few(hipStream_t st, const HeadArgs& g) {
  const int R = few_rows(g.M);
  const int lds = R * g.K * Types<TYPES>::kXBytes;
  const int waves = kFewThreads / 64;
  const int bands = g.N / 32;
  const int per_wave = ceil_div(bands, waves * device_cu_count());
  RWKV_HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void*>(head_few_kernel<TYPES>), hipFuncAttributeMaxDynamicSharedMemorySize, kFewLds));
  hipLaunchKernelGGL(head_few_kernel<TYPES>, dim3(ceil_div(bands, waves * per_wave)), dim3(kFewThreads), lds, st, g, __builtin_ctz(R), per_wave);
  RWKV_LAUNCH_CHECK();
  return RWKV_OK;
}

template <int TYPES, bool SUMS>
int launch_tiles(hipStream_t st, HeadArgs g) {
  const int rows = g.M <= 128 ? 128 : 256;
  g.row_tiles = ceil_div(g.M, rows);
  g.col_blocks = ceil_div(g.N, kTileCols);
  const dim3 grid(g.row_tiles * ceil_div(g.col_blocks, 8) * 8);
  if (rows == 256) hipLaunchKernelGGL((head_tile_kernel<TYPES, 4, SUMS>), grid, dim3(64 * kTileWaves), 0, st, g);
  else hipLaunchKernelGGL((head_tile_kernel<TYPES, 2, SUMS>), grid, dim3(64 * kTileWaves), 0, st, g);
  RWKV_LAUNCH_CHECK();
  return RWKV_OK;
}

template <int TYPES>
int launch_rows(hipStream_t st, const Plan& p, HeadArgs g, const TokenLogprobs& out, void* rest) {
  if (p.way == kSums) {
    const int rc = launch_tiles<TYPES, true>(st, g);
    if (rc != RWKV_OK) return rc;
    g.col_blocks = ceil_div(g.N, kTileCols);
    hipLaunchKernelGGL(head_join_kernel, dim3(ceil_div(g.M, 16)), dim3(256), 0, st, g, out);
    RWKV_LAUNCH_CHECK();
    return RWKV_OK;
  }
  const int rc = p.way == kFew ? launch_few<TYPES>(st, g) : launch_tiles<TYPES, false>(st, g);
  if (rc != RWKV_OK) return rc;
  return token_logprobs_launch(st, g.M, g.N, RWKV_IO_F32, g.logits, g.N, out, rest);
}

}  // namespace

size_t linear_logprobs_workspace_bytes(int fmt, bool x_int8, int M, int N, int K, int top_n) { return plan_of(x_int8, M, N, K, top_n).bytes(); }

int linear_logprobs_launch(hipStream_t st, int fmt, int M, int N, int K, const void* x, const float* x_scale, const void* packed,
                           const half_t* scale, const TokenLogprobs& out, void* workspace) {
  const Plan p = plan_of(x_scale != nullptr, M, N, K, out.top_n);
  unsigned char* ws = static_cast<unsigned char*>(workspace);
  for (int m = 0; m < M; m += p.rows) {
    const int64_t off = static_cast<int64_t>(m) * K * (x_scale ? 1 : 2);
    const TokenLogprobs rows = out.from_row(m);
    HeadArgs g = {static_cast<const char*>(x) + off, x_scale ? x_scale + m : nullptr, static_cast<const char*>(packed), scale,
                  std::min(p.rows, M - m), N, K, reinterpret_cast<float*>(ws), rows.logprob ? rows.tokens : nullptr,
                  reinterpret_cast<float4_t*>(ws + p.logits), reinterpret_cast<float*>(ws + p.logits + p.part), out.top_n == 1, 0, 0};
    void* rest = ws + p.logits + p.part + p.token_logit;
    const int rc = x_scale ? launch_rows<kI8W8>(st, p, g, rows, rest)
                           : (fmt == RWKV_FMT_W8 ? launch_rows<kF16W8>(st, p, g, rows, rest) : launch_rows<kF16F16>(st, p, g, rows, rest));
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
  RWKV_REQUIRE(N <= kMaxLogprobVocab && K <= kMaxHeadWidth, "%s: N up to %d and K up to %d, got %d and %d", who, kMaxLogprobVocab, kMaxHeadWidth, N, K);
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
