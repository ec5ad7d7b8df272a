// Tiles, stages and tensor memory of the microscaled products (ko_mx_gemm.cu), without anything of CUDA's, so that a host
// program can take them apart.
#pragma once

#include <cstddef>
#include <cstdint>

#include "ko_residency.h"

#if defined(__CUDACC__)
#define KO_HD __host__ __device__
#else
#define KO_HD
#endif

namespace komx {

template <bool F4>
struct Elem {
  static constexpr uint32_t kTypeA = F4 ? 1u : 0u;  // e2m1 / e4m3
  static constexpr uint32_t kTypeW = F4 ? 1u : 5u;  // e2m1 in either kind's numbering
  static constexpr int kStageK = F4 ? 256 : 128;    // elements along K per stage: 128 bytes of shared memory per row
  static constexpr int kKt = kStageK / 128;         // scale tiles along K per stage
  static constexpr int kMma = 4;                    // instructions along K per stage, 32 bytes each
  // What a barrier counts for a box of 128 weight rows: the bytes that TMA reads. A spread box reads half of what it fills.
  static constexpr uint32_t kTxW = 128 * (F4 ? 128 : 64);
  // scale word (tile along K) and first scale byte of instruction j
  static constexpr KO_HD int kt_of(int j) { return F4 ? j >> 1 : 0; }
  static constexpr KO_HD uint32_t sf_of(int j) { return F4 ? static_cast<uint32_t>(j & 1) * 2 : j; }
};

template <bool F4, int BN>
struct PairCfg {
  // Rows of the staging tiles: 128 bytes, or 64 where the room is better used for a stage more (BN 256: 8192 x 4096 x 8192
  // in mxfp8 in 185 us with five stages, in 193 with four and 128-byte rows).
  static constexpr int kRow = BN == 256 ? 64 : 128;
  static constexpr int kStages = BN == 256 ? 5 : 6;
  static constexpr uint32_t kA = 128 * 128, kW = BN / 2 * 128;
  static constexpr uint32_t kSfa = 512 * Elem<F4>::kKt, kSfw = BN / 128 * kSfa;
  static constexpr uint32_t kOffSf = kA + kW;
  static constexpr uint32_t kStage = (kOffSf + kSfa + kSfw + 1023) / 1024 * 1024;
  static constexpr uint32_t kTx = 2 * (kA + Elem<F4>::kTxW * BN / 256 + kSfa + kSfw);  // both CTAs
  static constexpr uint32_t kOffStaging = kStages * kStage;
  static constexpr uint32_t kStaging = 32 * kRow;  // 32 rows for each epilogue warp
  static constexpr uint32_t kOffBias = kOffStaging + 16 * kStaging;  // 64 columns for each epilogue warp
  static constexpr uint32_t kOffBars = kOffBias + 16 * 64 * 4;
  static constexpr uint32_t kSmem = 1024 + kOffBars + 256;
  static constexpr int kAccs = BN == 256 ? 2 : 3;                // accumulators, 128 columns apart
  static constexpr uint32_t kSfwCols = 4 * (BN / 128);
  static constexpr uint32_t kColSf = 384, kSfCols = (4 + kSfwCols) * Elem<F4>::kKt;  // a slot
  static_assert(BN == 128 || BN == 256, "tile width");
  static_assert(kSmem >= ko::kWholeTmemSmem, "a CTA with all of tensor memory has its SM to itself");
  static_assert(kColSf + kStages * kSfCols <= 512, "tensor memory");
  static_assert((2 * kStages + 2 * kAccs + 2) * 8 + 16 <= 256, "barrier area");
};

template <bool F4, int BN>
struct SliceCfg {
  static constexpr uint32_t kW = 128 * 128, kX = BN * 128, kSf = 512 * Elem<F4>::kKt;
  static constexpr uint32_t kOffSf = kW + kX;
  static constexpr uint32_t kStage = (kW + kX + 2 * kSf + 1023) / 1024 * 1024;
  static constexpr uint32_t kTx = Elem<F4>::kTxW + kX + 2 * kSf;
  static constexpr int kStages = BN <= 32 ? 5 : BN <= 64 ? 4 : 3;  // what half of an SM's shared memory holds
  static constexpr uint32_t kOffBars = kStages * kStage;
  static constexpr uint32_t kSmemNeed = 1024 + kOffBars + 256;
  // More than the stages need where these are few: two of these CTAs share an SM, and none shares one with a kernel that
  // takes all of its tensor memory.
  static constexpr uint32_t kSmem = kSmemNeed > ko::kHalfTmemSmem ? kSmemNeed : ko::kHalfTmemSmem;
  static constexpr uint32_t kAccCols = BN < 32 ? 32 : BN;
  static constexpr uint32_t kSfCols = 8 * Elem<F4>::kKt;
  static constexpr uint32_t kNeed = kAccCols + kStages * kSfCols;
  static constexpr uint32_t kCols = kNeed <= 64 ? 64 : kNeed <= 128 ? 128 : 256;
  static_assert(kNeed <= 256, "two CTAs of an SM share 512 columns");
  static_assert(2 * (kSmem + ko::kSmemPerCta) <= ko::kSmemPerSm, "two CTAs share an SM");
  static_assert(BN * 128 * 4 <= kOffBars, "partial sums reuse the stages");
  static_assert((2 * kStages + 1) * 8 + 16 <= 256, "barrier area");
};

}  // namespace komx
