// The main loop of the tiles of 256 columns: X and packed weights through a ring of LDS stages that every wavefront fills with
// direct-to-LDS loads (gemm_tile.hip: the packed product and what bounds it; linear_logprobs.hip: the head with its log probabilities).
#pragma once

#include "gemm_stream.h"

namespace rwkv {

typedef int int4v_t __attribute__((ext_vector_type(4)));
typedef int int16v_t __attribute__((ext_vector_type(16)));

constexpr int kTileWaves = 8;
constexpr int kTileRowBytes = 128;  // of X per stage: 64 k of fp16, 128 of int8
constexpr int kTileCols = 256;
constexpr int kTileI8 = 100;  // beside RWKV_FMT_F16 and RWKV_FMT_W8 (fp16 x): int8 x and int8 weights, products in whole numbers

template <int FMT, int MT>
struct WideTile {
  typedef std::conditional_t<FMT == kTileI8, int16v_t, float16_t> acc_t;
  static constexpr int kK = FMT == kTileI8 ? 128 : 64;  // k per stage
  static constexpr int BM = 64 * MT;  // wavefronts 2 (rows) x 4 (columns), each 32 MT x 64
  static constexpr int kXBytes = BM * kTileRowBytes;
  static constexpr int kPieces = FMT == RWKV_FMT_W8 ? 2 : 4;  // 1 KiB weight pieces of a band and stage
  static constexpr int kStageBytes = kXBytes + 8 * kPieces * 1024;
  static constexpr int kStages = kStageBytes <= 32768 ? 4 : (kStageBytes <= 49152 ? 3 : 2);
  static constexpr int kXLoads = BM / 8 / kTileWaves;   // 1 KiB direct-to-LDS loads per wavefront and stage
  static constexpr int kLoads = kXLoads + kPieces;
  static constexpr int kOutLd = 64 + 4;
  static constexpr int kOutBytes = kTileWaves * 32 * kOutLd * 4;  // the epilogue's 32 rows x 64 columns of every wavefront
  static constexpr int kLdsBytes = kStages * kStageBytes > kOutBytes ? kStages * kStageBytes : kOutBytes;
};

// 64 lanes x 16 bytes from base + off into LDS from `lds` on.  In asm, because the compiler would wait for every such load in flight
// at the next read of LDS.
template <bool ONCE = false>
__device__ __forceinline__ void load_to_lds(uint32_t lds, uint32_t off, const void* base) {
  if constexpr (ONCE) asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 nt" ::"{m0}"(lds), "v"(off), "s"(base) : "memory");
  else asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"{m0}"(lds), "v"(off), "s"(base) : "memory");
}

template <int N>
__device__ __forceinline__ void meet() {  // all but the N youngest loads of this wavefront have landed, its LDS reads are done
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// acc[nb][mt] = the 32 columns nb of this wavefront's 64 x the 32 rows mt of its 32 MT: lane (j, h) holds, of row j, columns
// 8 (v / 4) + 4 h + v % 4.  x_base: row 0 of the block's rows (`rows` of them exist; the others repeat the last one) at the first k;
// w_base: the same k of band `wave` of the block's eight bands of 32 columns.  nstages: of T::kK k, at least one.
// ONCE: no other block reads these weights (they are not kept in the caches).
template <int FMT, int MT, bool ONCE = false>
__device__ __forceinline__ void tile_products(const char* x_base, uint32_t x_row_bytes, int rows, const char* w_base, int nstages,
                                              unsigned char* lds, typename WideTile<FMT, MT>::acc_t (&acc)[2][MT]) {
  using T = WideTile<FMT, MT>;
  constexpr int S = T::kStages;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int lane = threadIdx.x & 63;
  const int j = lane & 31, h = lane >> 5;
  const int wm = wave & 1, wn = wave >> 1;

  // Loads of a stage: wavefront w brings rows 8 (8 i + w) .. + 7 of X and band w of the weights.  LDS receives lane after lane; the
  // 16-byte pieces of row r of X lie permuted by r & 7, so the permutation is in the addresses it reads from.
  uint32_t x_off[T::kXLoads];
#pragma unroll
  for (int i = 0; i < T::kXLoads; ++i) {
    const int r = (i * kTileWaves + wave) * 8 + (lane >> 3);
    const int row = r < rows ? r : rows - 1;  // rows past M repeat the last one (not stored)
    x_off[i] = static_cast<uint32_t>(row) * x_row_bytes + (((lane & 7) ^ (r & 7)) << 4);
  }
  const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) unsigned char*)lds));
  auto request_one = [&](int i, int c, int slot) {
    const uint32_t dst = lds0 + slot * T::kStageBytes;
    if (i < T::kXLoads) {
      load_to_lds(dst + (i * kTileWaves + wave) * 1024, x_off[i < T::kXLoads ? i : 0], x_base + c * kTileRowBytes);
    } else {
      const int q = i - T::kXLoads;
      load_to_lds<ONCE>(dst + T::kXBytes + (wave * T::kPieces + q) * 1024, lane * 16, w_base + (static_cast<int64_t>(c) * T::kPieces + q) * 1024);
    }
  };

#pragma unroll
  for (int nb = 0; nb < 2; ++nb)
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int v = 0; v < 16; ++v) acc[nb][mt][v] = 0;

  int x_at[4];  // of the MFMA steps (16 k of fp16, 32 of int8 each)
#pragma unroll
  for (int st = 0; st < 4; ++st) x_at[st] = wm * MT * 4096 + j * 128 + (((FMT == kTileI8 ? st * 2 + h : (st >> 1) * 4 + h * 2 + (st & 1)) ^ (j & 7)) << 4);
  const int w_at = T::kXBytes + wn * 2 * T::kPieces * 1024 + lane * 16;

  half8_t a[2][MT];
  uint4_t w[2][2];  // of two steps; int8 under fp16 x: of two 32-k groups, each two steps
  auto load_x = [&](const unsigned char* xs, int st, half8_t (&dst)[MT]) {
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) dst[mt] = *reinterpret_cast<const half8_t*>(xs + x_at[st] + mt * 4096);
  };
  auto load_w = [&](const unsigned char* xs, int piece, uint4_t (&dst)[2]) {
#pragma unroll
    for (int nb = 0; nb < 2; ++nb) dst[nb] = *reinterpret_cast<const uint4_t*>(xs + w_at + (nb * T::kPieces + piece) * 1024);
  };
  auto multiply = [&](int st) {
#pragma unroll
    for (int nb = 0; nb < 2; ++nb) {
      if constexpr (FMT == kTileI8) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
          acc[nb][mt] = __builtin_amdgcn_mfma_i32_32x32x32_i8(__builtin_bit_cast(int4v_t, w[st & 1][nb]), __builtin_bit_cast(int4v_t, a[st & 1][mt]),
                                                              acc[nb][mt], 0, 0, 0);
      } else {
        half8_t b;
        if constexpr (FMT == RWKV_FMT_F16) {
          b = __builtin_bit_cast(half8_t, w[st & 1][nb]);
        } else {
          const uint4_t& p = w[st >> 1][nb];
          b = st & 1 ? expand_w8(p[2], p[3]) : expand_w8(p[0], p[1]);
        }
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) acc[nb][mt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(b, a[st & 1][mt], acc[nb][mt], 0, 0, 0);
      }
    }
  };

#pragma unroll
  for (int c = 0; c < S - 1; ++c)
    if (c < nstages) {
#pragma unroll
      for (int i = 0; i < T::kLoads; ++i) request_one(i, c, c);
    }
  if (nstages >= S - 1) meet<T::kLoads * (S - 2)>();
  else meet<0>();
  load_x(lds, 0, a[0]);
  load_w(lds, 0, w[0]);

  int slot = 0, slot_free = S - 1;
  // Stage c; `more`: stage c + S - 1 exists and is requested, into the place of stage c - 1, which everybody has read.  The block meets
  // ahead of the last step, whose fragments are in registers by then: stage c + 1 has landed and its first ones are read under
  // that step's products.
  auto stage = [&](int c, auto more) {
    const unsigned char* xs = lds + slot * T::kStageBytes;
    slot = slot + 1 == S ? 0 : slot + 1;
    const unsigned char* xs_next = lds + slot * T::kStageBytes;
#pragma unroll
    for (int st = 0; st < 4; ++st) {
      if constexpr (decltype(more)::value) {
#pragma unroll
        for (int i = 0; i < T::kLoads; ++i)
          if (i * 3 / T::kLoads == st) request_one(i, c + S - 1, slot_free);
      }
      if (st < 3) {
        load_x(xs, st + 1, a[(st + 1) & 1]);
        if constexpr (FMT != RWKV_FMT_W8) load_w(xs, st + 1, w[(st + 1) & 1]);
        else if (st == 0) load_w(xs, 1, w[1]);
      } else {
        if constexpr (decltype(more)::value) meet<T::kLoads * (S - 2)>();
        else meet<0>();
        load_x(xs_next, 0, a[0]);
        if constexpr (FMT != RWKV_FMT_W8) load_w(xs_next, 0, w[0]);
      }
      __builtin_amdgcn_sched_barrier(0);
      multiply(st);
      if constexpr (FMT == RWKV_FMT_W8) {
        if (st == 3) load_w(xs_next, 0, w[0]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    slot_free = slot_free + 1 == S ? 0 : slot_free + 1;
  };
  int c = 0;
  for (; c + S - 1 < nstages; ++c) stage(c, std::true_type{});
  for (; c < nstages; ++c) stage(c, std::false_type{});  // (the last one reads on into a stage that is not multiplied)
  meet<0>();
}

}  // namespace rwkv
