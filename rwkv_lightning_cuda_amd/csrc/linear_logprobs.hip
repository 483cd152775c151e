// The vocabulary's product with the log probabilities of its logits: z[M,N] = x[M,K] . W[N,K]^T in fp32 (not rounded to fp16 as the
// logits of a forward pass are), then what logprobs.hip makes of the rows.  x fp16 with fp16 or int8 weights, or int8 codes with a
// scale per row and int8 weights (products in whole numbers, exact in 32 bits: 128 * 128 K < 2^31 up to K = 131071).
// Reference: the head product alone (src/rwkv7_fast_v4.cu:1325-1341).
#include <algorithm>
#include <utility>

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
  const int* tokens;     // may be NULL
  float4_t* sums;        // [M][parts]: m, S, U of a part's columns (few rows: a block's, tiles: 256)
  float* token_logit;    // [M], written where the token is a column
  int* firsts;           // one alternative from tiles: [M][parts], the first column of a part's largest logit; else NULL
  // alternatives only
  float* logits;         // [M,N], written where it may hold one
  float* strips;         // [M][4 parts]: largest of each 64 columns (tiles)
  const float* bound;    // [M] or NULL: strips below it are not written
  int parts, row_tiles;
  // which blocks of 256 columns a launch takes: block i is c = i * every, or with `rest` what is left out by that
  int col_blocks, every;
  bool rest;
};

// of two places the one with the larger value, the lower of equal ones
__device__ __forceinline__ int first_of(float m, int i, float o, int k) { return o > m ? k : o == m ? min(i, k) : i; }

// ---- few rows: the weights are streamed once, which is what bounds it ------------------------------------------------
// A wavefront takes whole bands of 32 columns, one after the other in memory, 8 KiB of them requested ahead of the 8 KiB that it
// multiplies.  x lies in LDS in the order in which the matrix core's lanes read it - lane (j, h) the 16 bytes of row j & (R - 1), k =
// 32 g + 16 h (int8) or + 8 i (fp16) - R = the rows rounded up to a power of two.  The weights are read once and not kept in the caches
// (non-temporal loads: one row of 4096 int8 58 -> 52 us, fp16 100 -> 88).  One row of 4096 int8, 65536 columns: 268 MB in 49 us of kernel,
// 5.5 TB/s (a large copy moves 4.9); two or three chunks in flight instead of one change it by 1 %.
constexpr int kFewThreads = 512;
constexpr int kFewLds = 128 * 1024;
constexpr int kFewRows = 32;  // rows of a product; us as tiles, 32 rows: 4096 int8 55 / 56 so, 2048 fp16 56 / 55, int8 weights under it 39 / 34, 768 fp16 29 / 23
constexpr int kFewMergeBytes = kFewThreads / 64 * kFewRows * 16;

int few_rows(int M) {
  int r = 1;
  while (r < M) r *= 2;
  return r;
}
// bands of 32 columns per wavefront: one round of blocks on the chip
int few_bands(int N) { return ceil_div(N / 32, kFewThreads / 64 * device_cu_count()); }
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
    for (int p = 0; p < kChunk; ++p) ahead[p] = __builtin_nontemporal_load(w + p * 64);
    w += kChunk * 64;
  };
  if (chunks > 0) request();
  // x: 16-byte piece n of row r (int8: of k = 16 n, the lanes' h is n % 2; fp16: of k = 8 n, h is the second bit of n, i the first)
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
  const int token = g.tokens ? g.tokens[min(j, g.M - 1)] : -1;
  typedef typename WideTile<T::kTile, 2>::acc_t acc_t;
  SoftSum total;
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
    float z[16];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      half4_t sc = {1, 1, 1, 1};
      if (TYPES != kF16F16) sc = *reinterpret_cast<const half4_t*>(g.scale + band * 32 + 8 * q + 4 * h);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        z[4 * q + i] = static_cast<float>(acc[4 * q + i]);
        if (TYPES != kF16F16) z[4 * q + i] = mul_f32(z[4 * q + i], h2f(sc[i]));
        if (TYPES == kI8W8) z[4 * q + i] = mul_f32(z[4 * q + i], xs);
      }
    }
    SoftSum a;
#pragma unroll
    for (int v = 0; v < 16; ++v) a.m = fmaxf(a.m, z[v]);
#pragma unroll
    for (int v = 0; v < 16; ++v) a.add(z[v]);
    total.merge(a);
    if (j < g.M) {
      const int t = token - band * 32 - 4 * h;
      if (t >= 0 && t < 32) {
#pragma unroll
        for (int v = 0; v < 16; ++v)
          if (t == 8 * (v >> 2) + (v & 3)) g.token_logit[j] = z[v];
      }
      if (g.logits) {
#pragma unroll
        for (int q = 0; q < 4; ++q)
          *reinterpret_cast<float4_t*>(g.logits + static_cast<int64_t>(j) * g.N + band * 32 + 8 * q + 4 * h) =
              float4_t{z[4 * q], z[4 * q + 1], z[4 * q + 2], z[4 * q + 3]};
      }
    }
  }
  // the block's columns
  total.merge_lanes<32>();
  __syncthreads();
  float4_t* merge = reinterpret_cast<float4_t*>(x_lds);  // [kWaves][kFewRows]
  if (h == 0 && j < g.M) merge[wave * kFewRows + j] = total.stored();
  __syncthreads();
  const int r = threadIdx.x;
  if (r < g.M) {
    SoftSum a;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) a.merge(SoftSum(merge[i * kFewRows + r]));
    g.sums[static_cast<int64_t>(r) * g.parts + blockIdx.x] = a.stored();
  }
}

// ---- many rows: the tiles of the packed product -----------------------------------------------------------------------
// A tile leaves m, S and U of its 256 columns for every row (16 bytes for 1 KiB of logits).  A lane has 32 columns of a row in
// registers: they are reduced there, with the other half's 32 by a swap of rows, with the other three wavefronts' 64 each through LDS.
// LOGITS: also the largest of each 64 columns, and the logits of those 64 where that is not below the row's bound.  ONE: one tile of
// rows, whose weights no other block reads.
// What bounds it: the chip's power, as the packed product (matrix core busy 51 % of the time at 1.95 GHz); the sums take about a tenth.
// 2048 rows of 4096 int8, 65536 columns: 499 to 522 us on several cards, 2.1 to 2.2 P operations/s (a plain product of 8192 x 8192 x 8192
// reaches 2.08); fp16 979 us, 1.12 PFLOP/s.  Through blocks of 256 rows of logits in memory the int8 case with 5 alternatives took 798 us, so 550.
template <int TYPES, int MT, bool LOGITS, bool ONE>
__global__ __launch_bounds__(64 * kTileWaves, 2) void head_tile_kernel(HeadArgs g) {
  typedef Types<TYPES> T;
  typedef WideTile<T::kTile, MT> W;
  __shared__ __align__(1024) unsigned char lds[W::kStages * W::kStageBytes];
  const int id = blockIdx.x;
  const int row_tile = (id >> 3) % g.row_tiles;
  const int index = (id / (8 * g.row_tiles)) * 8 + (id & 7);
  if (index >= g.col_blocks) return;
  const int col_block = g.rest ? index + index / (g.every - 1) + 1 : index * g.every;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int lane = threadIdx.x & 63, j = lane & 31, h = lane >> 5;
  const int wm = wave & 1, wn = wave >> 1;
  const int m0 = row_tile * W::BM;
  const int band = min(col_block * 8 + wave, g.N / 32 - 1);  // past the last band: repeat it
  typename W::acc_t acc[2][MT];
  tile_products<T::kTile, MT, ONE>(g.x + static_cast<int64_t>(m0) * g.K * T::kXBytes, static_cast<uint32_t>(g.K) * T::kXBytes, g.M - m0,
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
  float4_t* merge = reinterpret_cast<float4_t*>(lds);          // [4][BM]
  int* merge_first = reinterpret_cast<int*>(merge + 4 * W::BM);  // [4][BM]
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
    // m and U in units of x_scale, as everything up to the exponent
    SoftSum a;
#pragma unroll
    for (int nb = 0; nb < 2; ++nb)
      if (col0 + nb * 32 < g.N) {
#pragma unroll
        for (int v = 0; v < 16; ++v) a.m = fmaxf(a.m, z[nb][v]);
      }
    const float to_log2 = xs * kLog2e;
    float all = 0.0f;
#pragma unroll
    for (int nb = 0; nb < 2; ++nb)
      if (col0 + nb * 32 < g.N) {
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          const float d = z[nb][v] - a.m;
          const float p = __builtin_amdgcn_exp2f(d * to_log2);
          all += p;
          a.s += __builtin_amdgcn_fractf(p);  // (p, but for the largest ones' 1: as add() keeps them apart)
          a.u = fmaf(d, p, a.u);
        }
      }
    if (__any(a.u != a.u && all == all)) {  // a d of -infinity, whose p is 0
      a.u = 0.0f;
#pragma unroll
      for (int nb = 0; nb < 2; ++nb)
        if (col0 + nb * 32 < g.N) {
#pragma unroll
          for (int v = 0; v < 16; ++v) {
            const float d = z[nb][v] - a.m;
            a.u = fmaf(fmaxf(d, kLowest), __builtin_amdgcn_exp2f(d * to_log2), a.u);
          }
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
    if (TYPES == kI8W8 && a.m != kLowest) {  // (the lowest value stands for none)
      a.m *= xs;
      a.u *= xs;
    }
    a.n = rintf(all - a.s);
    int first = g.N;
    if (!LOGITS && g.firsts) {
#pragma unroll
      for (int nb = 1; nb >= 0; --nb)
        if (col0 + nb * 32 < g.N) {
#pragma unroll
          for (int v = 15; v >= 0; --v)
            if ((TYPES == kI8W8 ? mul_f32(z[nb][v], xs) : z[nb][v]) == a.m) first = col0 + 4 * h + nb * 32 + 8 * (v >> 2) + (v & 3);
        }
      first = first_of(a.m, first, lane_xor_f<32>(a.m), lane_xor_dpp<32>(first));
      if (h == 0) merge_first[wn * W::BM + r] = first;
    }
    a.merge_lanes<32>();
    if (h == 0) merge[wn * W::BM + r] = a.stored();
    if constexpr (LOGITS) {
      if (live && !(g.bound && a.m < g.bound[row])) {
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
      }
    }
  }
  __syncthreads();
  const int r = threadIdx.x;
  if (r < W::BM && m0 + r < g.M) {
    SoftSum a;
    float4_t most;
    int first = g.N;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float4_t o = merge[i * W::BM + r];
      most[i] = o[0];
      if (!LOGITS && g.firsts) first = first_of(a.m, first, o[0], merge_first[i * W::BM + r]);
      a.merge(SoftSum(o));
    }
    const int64_t at = static_cast<int64_t>(m0 + r) * g.parts + col_block;
    g.sums[at] = a.stored();
    if constexpr (LOGITS) *reinterpret_cast<float4_t*>(g.strips + at * 4) = most;
    else if (g.firsts) g.firsts[at] = first;
  }
}

// What the top_n-th largest of the strips that the first launch has left reaches, a wavefront per row: no alternative lies below it.
constexpr int kBoundStrips = 1024;
template <int N>
__global__ __launch_bounds__(256) void head_bound_kernel(HeadArgs g, int top_n, float* bound) {
  const int row = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (row >= g.M) return;
  const float* strips = g.strips + static_cast<int64_t>(row) * g.parts * 4;
  float v[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int k = i * 64 + lane;
    v[i] = k < 4 * g.col_blocks ? strips[(k >> 2) * g.every * 4 + (k & 3)] : -INFINITY;
  }
  const float found = wave_bound(v, top_n);
  if (lane == 0) bound[row] = found;
}

// Log probability and entropy from the parts' sums, and the one alternative that they name: a wavefront per row.
__global__ __launch_bounds__(256) void head_sums_kernel(HeadArgs g, TokenLogprobs out) {
  const int row = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= g.M) return;
  const int64_t at = static_cast<int64_t>(row) * g.parts;
  const int token = g.tokens ? g.tokens[row] : -1;
  const float token_logit = g.token_logit[row];  // (not written where there is no token)
  SoftSum a;
  int first = g.N;
  for (int i = threadIdx.x & 63; i < g.parts; i += 4 * 64) {
    float4_t p[4];  // requested together
    int f[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int k = min(i + q * 64, g.parts - 1);
      p[q] = g.sums[at + k];
      f[q] = g.firsts ? g.firsts[at + k] : g.N;
    }
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (i + q * 64 < g.parts) {
        first = first_of(a.m, first, p[q][0], f[q]);
        a.merge(SoftSum(p[q]));
      }
  }
  const float mine = a.m;
  a.merge_wave();
  first = wave_reduce_dpp(mine == a.m ? first : g.N, [](int x, int y) { return min(x, y); });
  if ((threadIdx.x & 63) != 0) return;
  write_logprobs(a, out, row, g.N, token, token_logit);
  if (out.top_n == 1) write_alternative(out, row, 0, a.m > kLowest && first < g.N ? key_of(a.m, first) : 0, a.m, a.log_sum());
}

// The same with the alternatives, a block per row: they lie in the strips whose largest reaches the top_n-th largest of 64 or 256 groups
// of strips - few more than top_n of them - whose logits are there.  1024 strips at a time (2048 rows of 1024 strips, 5 alternatives: 11 us; 256
// strips at a time 14) and 768 columns; the list never overflows, it is thinned out first.  Strips of `width` columns: 64 with their largest in `strips` (tiles), or a part's with it in `sums` (few rows).
__global__ __launch_bounds__(256) void head_alternatives_kernel(HeadArgs g, TokenLogprobs out, int width) {
  __shared__ __align__(16) Candidates<256> cand;
  __shared__ float4_t waves[4];
  constexpr int kStrips = 4;  // of a thread and turn
  __shared__ uint16_t chosen[kStrips * 256];  // (eight such blocks have room on a CU)
  static_assert(kMaxLogprobVocab / 64 <= 65536, "strips of 16 bits");
  __shared__ int n_chosen;
  const int tid = threadIdx.x, row = blockIdx.x, top_n = out.top_n;
  const float4_t* sums = g.sums + static_cast<int64_t>(row) * g.parts;
  const int n_strips = width == 64 ? 4 * g.parts : g.parts;
  const float* strips = width == 64 ? g.strips + static_cast<int64_t>(row) * n_strips : reinterpret_cast<const float*>(sums);
  const int apart = width == 64 ? 1 : 4;
  const float* logits = g.logits + static_cast<int64_t>(row) * g.N;
  const int token = g.tokens ? g.tokens[row] : -1;
  const float token_logit = g.token_logit[row];  // (not written where there is no token)
  float strip[kStrips];
  auto look = [&](int base) {
#pragma unroll
    for (int q = 0; q < kStrips; ++q) {
      const int s = base + q * 256 + tid;
      strip[q] = s < n_strips ? strips[s * apart] : -INFINITY;
    }
  };
  look(0);
  SoftSum a;
  for (int i = tid; i < g.parts; i += 256) a.merge(SoftSum(sums[i]));
  a.merge_wave();
  if ((tid & 63) == 0) waves[tid >> 6] = a.stored();
  if (tid == 0) {
    cand.n = 0;
    n_chosen = 0;
  }
  float most = -INFINITY;
#pragma unroll
  for (int q = 0; q < kStrips; ++q) most = fmaxf(most, strip[q]);
  for (int i = kStrips * 256 + tid; i < n_strips; i += 256) most = fmaxf(most, strips[i * apart]);
  // (not below the bound that the tiles went by: what lies below that has not been written)
  const float bound = fmaxf(first_bound(cand, top_n, most), g.bound ? g.bound[row] : -INFINITY);
  a = SoftSum();
#pragma unroll
  for (int i = 0; i < 4; ++i) a.merge(SoftSum(waves[i]));
  key_t least = bound == -INFINITY ? 0 : key_of(bound, 0x7fffffff);  // what a candidate has to be ahead of
  int list = 0;
  const int at_once = width < 256 ? width : 256;  // columns of a strip
  const int pieces = width / at_once;
  constexpr int kAtOnce = 3;
  static_assert(kMaxAlternatives <= kCandidates - kAtOnce * 256, "a list that has been thinned out takes the next entries");
  for (int base = 0; base < n_strips; base += kStrips * 256) {
    if (base > 0) look(base);
    // (a strip whose largest ties with the last candidate and lies behind it has none)
#pragma unroll
    for (int q = 0; q < kStrips; ++q) {
      const int s = base + q * 256 + tid;
      if (strip[q] > -INFINITY && key_of(strip[q], s * width) > least) chosen[atomicAdd(&n_chosen, 1)] = s;
    }
    __syncthreads();
    const int n = n_chosen * pieces;
    for (int k = 0; k < n; k += kAtOnce * (256 / at_once)) {
      float v[kAtOnce];
      int col[kAtOnce];
#pragma unroll
      for (int q = 0; q < kAtOnce; ++q) {  // requested together
        const int which = k + q * (256 / at_once) + tid / at_once;
        col[q] = which < n ? chosen[which / pieces] * width + which % pieces * at_once + tid % at_once : g.N;
        v[q] = col[q] < g.N ? logits[col[q]] : -INFINITY;
      }
#pragma unroll
      for (int q = 0; q < kAtOnce; ++q)
        if (v[q] > -INFINITY) {
          const key_t key = key_of(v[q], col[q]);
          if (key > least) offer(cand, list, key);
        }
      __syncthreads();
      const int have = cand.n;
      __syncthreads();
      if (have > kCandidates - kAtOnce * 256) {
        thin_out(cand, list, have, top_n);
        list ^= 1;
        __syncthreads();
        least = cand.list[list][top_n - 1];
        if (tid == 0) cand.n = top_n;
        __syncthreads();
      }
    }
    if (tid == 0) n_chosen = 0;
    __syncthreads();
  }
  const int n = cand.n;
  const float log_s = a.log_sum();
  thin_out(cand, list, n, top_n);
  __syncthreads();
  if (tid < top_n) write_alternative(out, row, tid, tid < n ? cand.list[list ^ 1][tid] : 0, a.m, log_s);
  if (tid == 0) write_logprobs(a, out, row, g.N, token, token_logit);
}

// ---- what a call takes ------------------------------------------------------------------------------------------------
struct Plan {
  bool few;
  int rows;        // at a time
  int tile;        // rows of a tile
  int parts;       // of a row, with sums of their own
  int every;       // > 1: a first launch takes every so many blocks of columns and bounds the alternatives of the others
  bool lists;      // alternatives out of strips of logits, not the one that the sums name
  size_t sums, token_logit, firsts, logits, strips, bound;  // bytes, in this order
  size_t bytes() const { return sums + token_logit + firsts + logits + strips + bound; }
};

constexpr int kSumRows = 8192;    // rows at a time without lists of alternatives, and
constexpr int kSums = 1 << 21;    // those times parts: 32 MiB of sums
constexpr int kLogits = 1 << 27;  // and with them, rows times columns: 512 MiB of places for logits, few of which are written
constexpr int kFewestTurns = 6;   // turns of blocks on the chip from which on two launches cost less than the logits they save

Plan plan_of(int fmt, bool x_int8, int M, int N, int K, int top_n) {
  Plan p = {};
  p.few = takes_few(M, K, x_int8 ? 1 : 2);
  p.lists = top_n > 1 || (top_n == 1 && p.few);
  p.parts = p.few ? ceil_div(N / 32, kFewThreads / 64 * few_bands(N)) : ceil_div(N, kTileCols);
  p.rows = p.few ? M : p.lists ? std::min(M, std::max(kLogits / N / 256, 1) * 256) : std::min({M, kSumRows, std::max(kSums / p.parts / 256, 1) * 256});
  // The tile whose rows, padding among them, cost least; a row of a lower tile costs more (us, 65536 columns, tiles of 128 / 192 / 256
  // rows: 768 rows of 2048 fp16 226 / 233 / 220, int8 weights under them 210 / 187 / 182, of 4096 int8 224 / 230 / 216; 333 rows 111 / 118 /
  // 136, 105 / 95 / 116, 113 / 120 / 137; 190 rows 77 / 67 / 75, 70 / 53 / 63, 80 / 68 / 78).
  const bool w8 = fmt == RWKV_FMT_W8 && !x_int8;
  int64_t least = INT64_MAX;
  for (const auto& [rows, cost] : {std::pair<int, int>{256, 100}, {192, w8 ? 104 : 112}, {128, w8 ? 122 : 106}}) {
    const int64_t all = static_cast<int64_t>(ceil_div(p.rows, rows)) * rows * cost;
    if (all >= least) continue;
    least = all;
    p.tile = rows;
  }
  p.every = 1;
  if (!p.few && p.lists) {
    const int64_t blocks = static_cast<int64_t>(ceil_div(p.rows, p.tile)) * p.parts, cus = device_cu_count();
    // (as many strips as groups of them are wanted, and no more than the bound's launch holds)
    if (blocks >= kFewestTurns * cus) p.every = std::min<int64_t>(ceil_div(blocks, cus), 4 * p.parts / std::max(2 * top_n, 128));
    if (p.every < 2 || 4 * ceil_div(p.parts, p.every) > kBoundStrips) p.every = 1;
  }
  const auto align = [](size_t n) { return (n + 255) / 256 * 256; };
  p.sums = align(static_cast<size_t>(p.rows) * p.parts * sizeof(float4_t));
  p.token_logit = align(static_cast<size_t>(p.rows) * 4);
  if (top_n == 1 && !p.lists) p.firsts = align(static_cast<size_t>(p.rows) * p.parts * sizeof(int));
  if (p.lists) p.logits = align(static_cast<size_t>(p.rows) * N * 4);
  if (p.lists && !p.few) p.strips = p.sums;
  if (p.lists && !p.few) p.bound = p.token_logit;  // (whether or not this call bounds them: fewer rows may)
  return p;
}

// of every call of up to M rows: fewer may go without tiles and keep all logits
size_t most_bytes(int fmt, bool x_int8, int M, int N, int K, int top_n) {
  int few = std::min(M, kFewRows);
  while (few > 0 && !takes_few(few, K, x_int8 ? 1 : 2)) --few;
  const size_t tiles = plan_of(fmt, x_int8, M, N, K, top_n).bytes();
  return few ? std::max(tiles, plan_of(fmt, x_int8, few, N, K, top_n).bytes()) : tiles;
}

template <int TYPES>
int launch_few(hipStream_t st, const HeadArgs& g) {
  const int R = few_rows(g.M);
  const int lds = std::max(R * g.K * Types<TYPES>::kXBytes, kFewMergeBytes);
  RWKV_HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void*>(head_few_kernel<TYPES>), hipFuncAttributeMaxDynamicSharedMemorySize, kFewLds));
  hipLaunchKernelGGL(head_few_kernel<TYPES>, dim3(g.parts), dim3(kFewThreads), lds, st, g, __builtin_ctz(R), few_bands(g.N));
  RWKV_LAUNCH_CHECK();
  return RWKV_OK;
}

// `col_blocks` of g.parts blocks of columns: every `every`-th, or the rest
template <int TYPES, bool LOGITS>
int launch_tiles(hipStream_t st, HeadArgs& g, int tile, int every, bool rest) {
  g.row_tiles = ceil_div(g.M, tile);
  g.every = every;
  g.rest = rest;
  g.col_blocks = rest ? g.parts - ceil_div(g.parts, every) : ceil_div(g.parts, every);
  const dim3 grid(g.row_tiles * ceil_div(g.col_blocks, 8) * 8);
  const bool one = g.row_tiles == 1;
  const auto kernel = tile == 256 ? (one ? head_tile_kernel<TYPES, 4, LOGITS, true> : head_tile_kernel<TYPES, 4, LOGITS, false>)
                    : tile == 192 ? (one ? head_tile_kernel<TYPES, 3, LOGITS, true> : head_tile_kernel<TYPES, 3, LOGITS, false>)
                                  : (one ? head_tile_kernel<TYPES, 2, LOGITS, true> : head_tile_kernel<TYPES, 2, LOGITS, false>);
  hipLaunchKernelGGL(kernel, grid, dim3(64 * kTileWaves), 0, st, g);
  RWKV_LAUNCH_CHECK();
  return RWKV_OK;
}

template <int TYPES>
int launch_rows(hipStream_t st, const Plan& p, HeadArgs g, const TokenLogprobs& out, float* bound) {
  int rc = RWKV_OK;
  if (p.few) {
    rc = launch_few<TYPES>(st, g);
  } else if (!p.lists) {
    rc = launch_tiles<TYPES, false>(st, g, p.tile, 1, false);
  } else {
    rc = launch_tiles<TYPES, true>(st, g, p.tile, p.every, false);
    if (rc == RWKV_OK && p.every > 1) {
      const dim3 grid(ceil_div(g.M, 4));
      if (4 * g.col_blocks <= 128) hipLaunchKernelGGL(head_bound_kernel<2>, grid, dim3(256), 0, st, g, out.top_n, bound);
      else hipLaunchKernelGGL(head_bound_kernel<kBoundStrips / 64>, grid, dim3(256), 0, st, g, out.top_n, bound);
      RWKV_LAUNCH_CHECK();
      g.bound = bound;
      rc = launch_tiles<TYPES, true>(st, g, p.tile, p.every, true);
    }
  }
  if (rc != RWKV_OK) return rc;
  if (!p.lists) hipLaunchKernelGGL(head_sums_kernel, dim3(ceil_div(g.M, 4)), dim3(256), 0, st, g, out);
  else hipLaunchKernelGGL(head_alternatives_kernel, dim3(g.M), dim3(256), 0, st, g, out, p.few ? few_bands(g.N) * (kFewThreads / 64 * 32) : 64);
  RWKV_LAUNCH_CHECK();
  return RWKV_OK;
}

}  // namespace

size_t linear_logprobs_workspace_bytes(int fmt, bool x_int8, int M, int N, int K, int top_n) { return most_bytes(fmt, x_int8, M, N, K, top_n); }

int linear_logprobs_launch(hipStream_t st, int fmt, int M, int N, int K, const void* x, const float* x_scale, const void* packed,
                           const half_t* scale, const TokenLogprobs& out, void* workspace) {
  const Plan p = plan_of(fmt, x_scale != nullptr, M, N, K, out.top_n);
  unsigned char* ws = static_cast<unsigned char*>(workspace);
  for (int m = 0; m < M; m += p.rows) {
    const int64_t off = static_cast<int64_t>(m) * K * (x_scale ? 1 : 2);
    const TokenLogprobs rows = out.from_row(m);
    HeadArgs g = {};
    g.x = static_cast<const char*>(x) + off;
    g.x_scale = x_scale ? x_scale + m : nullptr;
    g.wp = static_cast<const char*>(packed);
    g.scale = scale;
    g.M = std::min(p.rows, M - m);
    g.N = N;
    g.K = K;
    g.tokens = rows.logprob ? rows.tokens : nullptr;
    g.parts = p.parts;
    unsigned char* at = ws;
    const auto take = [&at](size_t bytes) {
      void* p = bytes ? at : nullptr;
      at += bytes;
      return p;
    };
    g.sums = static_cast<float4_t*>(take(p.sums));
    g.token_logit = static_cast<float*>(take(p.token_logit));
    g.firsts = static_cast<int*>(take(p.firsts));
    g.logits = static_cast<float*>(take(p.logits));
    g.strips = static_cast<float*>(take(p.strips));
    float* bound = static_cast<float*>(take(p.bound));
    const int rc = x_scale ? launch_rows<kI8W8>(st, p, g, rows, bound)
                           : (fmt == RWKV_FMT_W8 ? launch_rows<kF16W8>(st, p, g, rows, bound) : launch_rows<kF16F16>(st, p, g, rows, bound));
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
  const size_t need = plan_of(fmt, x_scale != nullptr, M, N, K, top_n).bytes();
  RWKV_REQUIRE(workspace && workspace_bytes >= need && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0,
               "linear_logprobs: workspace of %zu bytes (aligned to 16) needed, got %zu", need, workspace_bytes);
  return linear_logprobs_launch(as_stream(s), fmt, M, N, K, x, static_cast<const float*>(x_scale), packed, static_cast<const half_t*>(scale), out,
                                workspace);
}

}  // extern "C"
