// Packed-weight MFMA GEMM for many rows of int8 and fp16 weights: blocks of 256 or 128 rows x 256 columns, X and the weights through a
// ring of LDS stages that every wavefront fills with direct-to-LDS loads.
//
// Reference: as gemm_stream.hip (cuda/rwkv7_v3a_ops.cu:2235-2368).
//
// What bounds it: the power the chip may draw.  At 2048 rows the 256-row blocks take 2610 clocks per stage of 64 k - 2048 of them the
// matrix core's - at 1.6 GHz; half as many blocks, alone on half the CUs, as many clocks at 2.1-2.3 GHz.  So a block moves as few bytes
// per product as its registers allow:
//   * Eight wavefronts, two per SIMD, each 128 (64) rows x 64 columns of accumulators: an X fragment out of LDS feeds two MFMAs, a
//     weight fragment four (two).  Wavefronts of 256 x 64, one per SIMD, expand every int8 code once instead of twice and read a tenth
//     less from LDS, and were slower (16384 x 4096, 2048 rows: 250 us against 237): nothing fills their waits.
//   * X and weights go from memory to LDS without passing through registers, two or three stages ahead, and weights arrive in the
//     order in which the matrix core reads them.  One barrier per stage, ahead of the last of its four steps.
//   * int8 codes become fp16 in eight instructions per fragment (expand_w8).
// us per launch, weights in no cache, before (the register-staged 128 x 256 tile, one wavefront per SIMD) -> now:
//   int8, 2048 rows: 16384 x 4096 282 -> 236 (1.16 PFLOP/s), 12288 x 4096 244 -> 204, 4096 x 16384 297 -> 235, 4096 x 4096 85 -> 71
//   int8, 512 rows: 16384 x 4096 85 -> 70, 12288 x 4096 78 -> 60      fp16, 2048 rows: 16384 x 4096 305 -> 250, 8192 x 2048 95 -> 67
//   fp16, 999 rows: 8192 x 2048 45 -> 38, 6144 x 2048 41 -> 35
#include "gemm_tile.h"

namespace rwkv {

namespace {

template <int FMT, int MT>
__device__ __forceinline__ void tile_block(const StreamArgs& g, const StreamProblem& pr, int row_tile, int col_block, int split,
                                           unsigned char* lds) {
  using T = WideTile<FMT, MT>;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int lane = threadIdx.x & 63;
  const int j = lane & 31, h = lane >> 5;
  const int wm = wave & 1, wn = wave >> 1;
  const int m0 = row_tile * T::BM;
  const int kbeg = split * g.k_per_split;
  const int nstages = g.k_per_split / T::kK;

  // this lane's columns of the epilogue and their int8 scales
  const bool partial_out = g.splits > 1;
  const int col = col_block * kTileCols + wn * 64 + (lane & 7) * 8;
  half8_t scale_h;
#pragma unroll
  for (int e = 0; e < 8; ++e) scale_h[e] = static_cast<half_t>(1.0f);
  if (FMT == RWKV_FMT_W8 && !partial_out) scale_h = *reinterpret_cast<const half8_t*>(pr.scale + (col < pr.N ? col : pr.N - 8));

  const char* x_base = reinterpret_cast<const char*>(pr.x + static_cast<int64_t>(m0) * g.K + kbeg);
  const int band_here = col_block * 8 + wave;
  const int band = band_here * 32 < pr.N ? band_here : pr.N / 32 - 1;  // past the last band: repeat it (columns not stored)
  const char* w_base = reinterpret_cast<const char*>(pr.wp) +
                       (static_cast<int64_t>(band) * (g.K / 32) + kbeg / 32) * (T::kPieces / 2 * 1024);
  float16_t acc[2][MT];
  tile_products<FMT, MT>(x_base, static_cast<uint32_t>(g.K) * 2u, g.M - m0, w_base, nstages, lds, acc);

  // 32 rows x 64 columns of a wavefront at a time through its own part of LDS, written in 16/32-byte pieces along the rows
  float* out = reinterpret_cast<float*>(lds) + wave * 32 * T::kOutLd;
  float* part_out = partial_out ? pr.partial + static_cast<int64_t>(split) * g.M * pr.N : nullptr;
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
    for (int nb = 0; nb < 2; ++nb)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *reinterpret_cast<float4_t*>(out + j * T::kOutLd + nb * 32 + 8 * q + 4 * h) =
            float4_t{acc[nb][mt][4 * q], acc[nb][mt][4 * q + 1], acc[nb][mt][4 * q + 2], acc[nb][mt][4 * q + 3]};
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = i * 8 + (lane >> 3);
      const int row = m0 + (wm * MT + mt) * 32 + r;
      const float4_t lo = *reinterpret_cast<const float4_t*>(out + r * T::kOutLd + (lane & 7) * 8);
      const float4_t hi = *reinterpret_cast<const float4_t*>(out + r * T::kOutLd + (lane & 7) * 8 + 4);
      if (row >= g.M || col >= pr.N) continue;
      float val[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
      if (!partial_out) {
#pragma unroll
        for (int e = 0; e < 8; ++e) val[e] = finish_value(mul_f32(val[e], h2f(scale_h[e])), g.epilogue);
      }
      const int64_t o = static_cast<int64_t>(row) * pr.N + col;
      if (partial_out || g.out_f32) {
        float* dst = partial_out ? part_out + o : static_cast<float*>(pr.y) + o;
        *reinterpret_cast<float4_t*>(dst) = float4_t{val[0], val[1], val[2], val[3]};
        *reinterpret_cast<float4_t*>(dst + 4) = float4_t{val[4], val[5], val[6], val[7]};
      } else {
        half8_t hv;
#pragma unroll
        for (int e = 0; e < 8; ++e) hv[e] = f2h(val[e]);
        *reinterpret_cast<half8_t*>(static_cast<half_t*>(pr.y) + o) = hv;
      }
    }
    __builtin_amdgcn_wave_barrier();
  }
}

template <int MT>
__global__ __launch_bounds__(64 * kTileWaves, 2) void gemm_tile_kernel(StreamArgs g) {
  constexpr int kA = WideTile<RWKV_FMT_W8, MT>::kLdsBytes, kB = WideTile<RWKV_FMT_F16, MT>::kLdsBytes;
  __shared__ __align__(1024) unsigned char lds[kA > kB ? kA : kB];
  ride_along_copy(g.copy, gridDim.x, blockDim.x);
  const int id = blockIdx.x;
  const int row_tile = (id >> 3) % g.row_tiles;
  const int pair = (id / (8 * g.row_tiles)) * 8 + (id & 7);
  if (pair >= g.col_blocks * g.splits) return;
  const int col_all = pair % g.col_blocks;
  const int split = pair / g.col_blocks;
  int pi = 0;
  while (pi + 1 < g.n_problems && col_all >= g.block_end[pi]) ++pi;
  const int col_block = col_all - (pi > 0 ? g.block_end[pi - 1] : 0);
  const StreamProblem& pr = g.p[pi];
  if (pr.fmt == RWKV_FMT_W8) tile_block<RWKV_FMT_W8, MT>(g, pr, row_tile, col_block, split, lds);
  else tile_block<RWKV_FMT_F16, MT>(g, pr, row_tile, col_block, split, lds);
}

}  // namespace

int gemm_tile_launch(hipStream_t st, int rows, const StreamArgs& g) {
  const dim3 grid(g.row_tiles * ceil_div(g.col_blocks * g.splits, 8) * 8);
  if (rows == 256) hipLaunchKernelGGL(gemm_tile_kernel<4>, grid, dim3(64 * kTileWaves), 0, st, g);
  else hipLaunchKernelGGL(gemm_tile_kernel<2>, grid, dim3(64 * kTileWaves), 0, st, g);
  RWKV_LAUNCH_CHECK();
  return RWKV_OK;
}

}  // namespace rwkv
