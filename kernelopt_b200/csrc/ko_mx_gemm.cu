// Product of microscaled operands:  out[M][N] = act(A[M][K] @ W[N][K]^T + bias),  A in mxfp4 or mxfp8, W in mxfp4.
// Formats and layout: ko_mx.cuh.
//
// The 5th-generation tensor cores multiply the codes and apply both blocks' scales in the same instruction
// (tcgen05.mma ... block_scale), accumulating in fp32 in tensor memory:
//   A in mxfp4: kind::mxf4, 64 elements along K per instruction, both operands packed two per byte
//   A in mxfp8: kind::mxf8f6f4, 32 elements along K per instruction; the 4-bit weight stays packed in HBM and TMA spreads
//               it to one element per byte in shared memory, as that kind reads it
// An operand row is 128 bytes of shared memory per pipeline stage (256 mxfp4 or 128 mxfp8 elements), 128-byte swizzled. The
// scales of 128 rows x 128 elements are one 512-byte tile in HBM; TMA brings the stage's tiles in and tcgen05.cp spreads
// them over tensor memory, ahead of the stage's MMAs on the same pipe.
//
// Two kernels: pairs of CTAs with tiles of 256 rows for many rows (pair_kernel), and single CTAs over slices of K for few
// (slice_kernel); launch() says which takes a product. Every wait on a barrier in shared memory is bounded; one that runs out
// ends the kernel with KO_ERR_DEVICE_TIMEOUT in *dev_status. The allocation of tensor memory and the cluster's own barrier have
// no limit: ko_residency.h keeps the first from waiting for another kernel.
#include <algorithm>
#include <atomic>
#include <climits>
#include <string>
#include <type_traits>

#include "ko_mx.cuh"
#include "ko_mx_cfg.h"

namespace {

using namespace kodev;
using namespace komx;

// ---- tcgen05 block-scaled forms (PTX ISA, tcgen05.mma / tcgen05.cp) ----------------------------------------

// Instruction descriptor of the block-scaled kinds: element types at bits 7 and 10 (e2m1 is 1 in kind::mxf4 and 5 in
// kind::mxf8f6f4, e4m3 is 0), N / 8 at bit 17, e8m0 scales at bit 23, M / 128 at bit 27. The scale bytes that an
// instruction uses within its 32-bit scale word start at byte `sf`, given for A at bit 29 and for B at bit 4.
__host__ __device__ constexpr uint32_t idesc_bs(uint32_t a_type, uint32_t b_type, int m, int n) {
  return (a_type << 7) | (b_type << 10) | (static_cast<uint32_t>(n >> 3) << 17) | (1u << 23) |
         (static_cast<uint32_t>(m >> 7) << 27);
}
__host__ __device__ constexpr uint32_t idesc_sf(uint32_t sf) { return (sf << 29) | (sf << 4); }

// One elected lane issues; GROUP: CTAs whose tensor cores run the instruction as one.
template <int GROUP, bool F4>
__device__ __forceinline__ void mma_bs_w(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                         uint32_t accumulate) {
#define KO_MMA_BS(FORM)                                                                                        \
  asm volatile("{\n\t.reg .pred p, e;\n\tsetp.ne.b32 p, %6, 0;\n\telect.sync _|e, 0xffffffff;\n\t"             \
               "@e tcgen05.mma." FORM " [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),                       \
               "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)                                 \
               : "memory")
  if constexpr (GROUP == 2 && F4) KO_MMA_BS("cta_group::2.kind::mxf4.block_scale.scale_vec::2X");
  else if constexpr (GROUP == 2) KO_MMA_BS("cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X");
  else if constexpr (F4) KO_MMA_BS("cta_group::1.kind::mxf4.block_scale.scale_vec::2X");
  else KO_MMA_BS("cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X");
#undef KO_MMA_BS
}

// 512 bytes of shared memory (32 rows of 16 bytes) to four tensor-memory columns, the same in all four lane quarters. With
// GROUP 2 both CTAs of the pair copy, each from its own shared memory.
template <int GROUP>
__device__ __forceinline__ void cp_scales_w(uint32_t taddr, uint64_t desc) {
  if constexpr (GROUP == 2)
    asm volatile("{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
                 "@e tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;\n\t}" ::"r"(taddr), "l"(desc) : "memory");
  else
    asm volatile("{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
                 "@e tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;\n\t}" ::"r"(taddr), "l"(desc) : "memory");
}
// Shared-memory descriptor of a scale tile: no swizzle, 8-row groups of 16-byte rows 128 bytes apart.
__device__ __forceinline__ uint64_t scale_desc(uint32_t addr) {
  return static_cast<uint64_t>((addr >> 4) & 0x3FFFu) | (static_cast<uint64_t>(128u >> 4) << 16) |
         (static_cast<uint64_t>(128u >> 4) << 32) | (static_cast<uint64_t>(1u) << 46);
}

// TMA load into this CTA's shared memory whose bytes count on a barrier of the pair's leader (`bar`: shared::cluster).
__device__ __forceinline__ void tma_load_2d_pair(const CUtensorMap* map, uint32_t bar, void* dst, int32_t c0, int32_t c1) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%3, %4}], "
      "[%2];" ::"r"(smem_addr(dst)),
      "l"(map), "r"(bar), "r"(c0), "r"(c1)
      : "memory");
}
__device__ __forceinline__ float4 cluster_load_f4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}
// Arrive on a barrier of the pair's leader. What the arrival orders are tensor-memory reads, before the MMAs that the leader
// issues next, and the tcgen05 fences on both sides see to that; a release at cluster scope, a memory barrier across the
// pair, made each tile's hand-over half a microsecond longer (25664 x 128 x 1536 28.4 -> 20.8 us).
__device__ __forceinline__ void arrive_leader(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}

// ---- activation ----
// Two fp32 values in one 64-bit register: Blackwell's packed multiply and fused multiply-add.
__device__ __forceinline__ uint64_t pack_f2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpack_f2(uint64_t v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t mul_f2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t fma_f2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

// GELU of two values: v Phi(v) = max(v, 0) - |v| q with q = erfc(|v| / sqrt 2) / 2 = exp(-v^2 / 2) g(|v|). g is smooth
// on [0, 6] (it falls from 1/2 to 0.065), so a polynomial of degree 12 in |v| / 3 - 1 has it. Its fit is minimax (Lawson's
// weights) in what counts of g's error: |v| q is within 7e-8, for small |v| within 2.4e-7 |v|, so that small results keep their
// digits, and q within 2.4e-5 of itself, so that those on the negative side do. Least squares alone, with the same error of g
// everywhere, had 2.4e-6 |v| next to zero. Beyond 6, |v| g(|v|) stays at 6 g(6) = 0.389, on its way to 1 / sqrt(2 pi) = 0.399:
// results that are below 6e-9 there come out too small in magnitude, by 0.7 % at -7, 1.4 % at -9, 2 % at -13 and less than 2.6 %
// anywhere, and 0 below -13.2, where the exponential leaves the normal fp32 numbers. NaN stays NaN, and GELU(-inf) is 0, its
// limit.
// It costs one special-function instruction, and all else but the ends is packed: 25664 x 384 x 1536 with fp32 outputs takes
// 34 us without an activation and 41 with this one. A&S 7.1.26 as the fp32-grade GEMM has it (two special-function
// instructions, not packed) added 30 us to the same product at an earlier state of the epilogue.
__device__ __forceinline__ void gelu_pair(float& a, float& b) {
  constexpr float g[13] = {-0.12151453644037247f, 0.10321106761693954f, -0.0823381170630455f, 0.06228569149971008f,
                           -0.04591979831457138f, 0.03130459412932396f, -0.01686754636466503f, 0.01429088693112135f,
                           -0.01651555486023426f, 0.0023183149751275778f, 0.005299349781125784f, 0.0041989353485405445f,
                           -0.004534068051725626f};
  const uint64_t ax = pack_f2(fminf(fabsf(a), 6.f), fminf(fabsf(b), 6.f));
  const uint64_t s = fma_f2(ax, pack_f2(1.f / 3.f, 1.f / 3.f), pack_f2(-1.f, -1.f));
  uint64_t p = pack_f2(g[12], g[12]);
#pragma unroll
  for (int i = 11; i >= 0; --i) p = fma_f2(p, s, pack_f2(g[i], g[i]));
  const uint64_t v = pack_f2(a, b);
  float wa, wb, ma, mb;  // exp(-v^2 / 2) as 2^(-v^2 log2(e) / 2)
  unpack_f2(mul_f2(mul_f2(v, v), pack_f2(-0.7213475204444817f, -0.7213475204444817f)), wa, wb);
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(wa) : "f"(wa));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(wb) : "f"(wb));
  asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(ma) : "f"(a));
  asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(mb) : "f"(b));
  unpack_f2(fma_f2(ax, mul_f2(p, pack_f2(wa, wb)), pack_f2(ma, mb)), a, b);
}
template <int N>
__device__ __forceinline__ void apply_act(float (&v)[N], int act) {
  if (act == KO_ACT_GELU) {
#pragma unroll
    for (int i = 0; i < N; i += 2) gelu_pair(v[i], v[i + 1]);
  } else if (act == KO_ACT_RELU) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = v[i] < 0.f ? 0.f : v[i];  // NaN stays
  }
}

// ---------------------------------------------------------------------------------------------------------
// pair_kernel: persistent CTA pairs (clusters of two), 256 x BN output tiles. The pair's tensor cores run as one
// (cta_group::2): each CTA holds 128 rows of A and half of the BN weight rows of a stage and receives its 128 x BN half of
// the product in its own tensor memory, so an SM loads less per MMA than with tiles of its own.
//   warp 0       TMA producer of this CTA; its bytes count on the leader's `full` barrier
//   warp 1       tensor memory; in the leader it copies the scales and issues the MMAs of both CTAs
//   warps 2-17   epilogue, 64 columns of a lane quarter each: accumulator -> + bias, activation, one rounding -> a
//                swizzled tile in shared memory -> TMA store (rows of `out` on 16 bytes), or element stores (other N)
// Tensor memory (512 columns): the accumulators in [0, 384), the scales in [384, 512) with a slot per stage.
//   BN 256: two accumulators that share [128, 256). Warps 2-9 read the shared half into registers and then let the next
//           tile's MMAs go; warps 10-17 have until the tile after it for the other half.
//   BN 128: three accumulators; warps 2-9 take the even tiles and warps 10-17 the odd ones, so the MMAs run up to three
//           tiles ahead.
// The 576 threads leave 96 registers each: tiles of 256 spill 8 to 24 bytes, those of 128 with fp32 outputs 16 to 48.
// Measured: 8192 x 4096 x 8192 with bf16 outputs in 110 us in mxfp4 (5.0 PFLOP/s, tensor pipe 62 % busy, 9.6 TB/s from L2) and
// in 185 us in mxfp8 (3.0 PFLOP/s, 78 %); 25664 x 384 x 1536 with fp32 outputs in 35 us (4.5 TB/s written), 44 with GELU.
// ---------------------------------------------------------------------------------------------------------
constexpr int kPairThreads = 18 * 32;

struct PairArgs {
  const float* bias;
  void* out;
  int* dev_status;
  int64_t M, N;
  int act, k_stages, m_tiles, n_tiles, n_pairs, tma_out;
};

template <bool F4, int BN, typename T>
__global__ void __launch_bounds__(kPairThreads, 1)
    pair_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_w,
                const __grid_constant__ CUtensorMap map_sa, const __grid_constant__ CUtensorMap map_sw,
                const __grid_constant__ CUtensorMap map_out, const PairArgs a) {
  using C = PairCfg<F4, BN>;
  using E = Elem<F4>;
  constexpr int NA = C::kAccs;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::kOffBars);  // stage landed in both CTAs (leader: 1 + tx)
  uint64_t* empty = full + C::kStages;    // stage's MMAs done            (1 commit, both CTAs)
  // A barrier's parity cannot tell a phase from the one after the next, so every accumulator has barriers of its own: the
  // waiters of one are never two of its tiles behind.
  uint64_t* acc_full = empty + C::kStages;  // tile's MMAs done           (1 commit, both CTAs) x NA
  uint64_t* acc_free = acc_full + NA;     // read, but for a shared half  (8 warps x 2 CTAs, leader) x NA
  uint64_t* shared_free = acc_free + NA;  // shared half read             (8 warps x 2 CTAs, leader)
  uint64_t* mma_done = shared_free + 1;   // every MMA done               (1 commit, both CTAs)
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(mma_done + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const int pair = static_cast<int>(blockIdx.x >> 1);
  const int total = a.m_tiles * a.n_tiles;
  // Tiles in bands of eight row tiles, rows fastest: the pairs that run together share few strips of A and W.
  auto tile_at = [&](int t, int& m, int& n) {
    const int band = t / (8 * a.n_tiles), in = t - band * 8 * a.n_tiles;
    const int rows = min(8, a.m_tiles - band * 8);
    n = in / rows;
    m = band * 8 + (in - n * rows);
  };

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int i = 0; i < NA; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_free[i], 16);
    }
    mbar_init(shared_free, 16);
    mbar_init(mma_done, 1);
    *abort_flag = 0;
    fence_barrier_init();
    prefetch_tmap(&map_a);
    prefetch_tmap(&map_w);
    prefetch_tmap(&map_sa);
    prefetch_tmap(&map_sw);
    prefetch_tmap(&map_out);
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, 512);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // both CTAs' barriers are initialised before any arrival from the peer
  tc_fence_after();
  wait_for_previous_grid();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    if (lane == 0) {
      int st = 0;
      uint32_t phase = 0;
      bool ok = true;
      const uint32_t leader_full = cluster_map(smem_addr(full), 0);
      for (int t = pair; t < total && ok; t += a.n_pairs) {
        int mt, nt;
        tile_at(t, mt, nt);
        for (int ks = 0; ks < a.k_stages; ++ks) {
          if (!mbar_wait(&empty[st], phase ^ 1u, abort_flag)) {
            ok = false;
            break;
          }
          uint8_t* s = smem + st * C::kStage;
          const uint32_t bar = leader_full + st * 8;
          if (rank == 0) mbar_arrive_expect_tx(&full[st], C::kTx);
          const int r = static_cast<int>(rank);
          tma_load_2d_pair(&map_a, bar, s, ks * 128, mt * 256 + r * 128);
          tma_load_2d_pair(&map_w, bar, s + C::kA, ks * 128, nt * BN + r * (BN / 2));
          tma_load_2d_pair(&map_sa, bar, s + C::kOffSf, ks * 64 * E::kKt, mt * 2 + r);
          tma_load_2d_pair(&map_sw, bar, s + C::kOffSf + C::kSfa, ks * 64 * E::kKt, nt * (BN / 128));
          if (++st == C::kStages) {
            st = 0;
            phase ^= 1u;
          }
        }
      }
    }
  } else if (warp == 1) {
    if (rank == 0) {
      constexpr uint32_t idesc = idesc_bs(E::kTypeA, E::kTypeW, 256, BN);
      const uint32_t sb = smem_addr(smem);
      int st = 0, local = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int t = pair; t < total && ok; t += a.n_pairs, ++local) {
        const int buf = local % NA, use = local / NA;  // this tile's accumulator, and the tiles before it there
        if (BN == 256 && local > 0 && !mbar_wait_warp(shared_free, static_cast<uint32_t>(local - 1) & 1u, abort_flag))
          break;
        if (use > 0 && !mbar_wait_warp(&acc_free[buf], static_cast<uint32_t>(use - 1) & 1u, abort_flag)) break;
        tc_fence_after();
        const uint32_t d = tmem + buf * 128;
        for (int ks = 0; ks < a.k_stages; ++ks) {
          if (!mbar_wait_warp(&full[st], phase, abort_flag)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t s = sb + st * C::kStage;
          const uint32_t sfa = tmem + C::kColSf + st * C::kSfCols, sfw = sfa + 4 * E::kKt;
#pragma unroll
          for (int kt = 0; kt < E::kKt; ++kt) {
            cp_scales_w<2>(sfa + 4 * kt, scale_desc(s + C::kOffSf + kt * 512));
#pragma unroll
            for (int i = 0; i < BN / 128; ++i)
              cp_scales_w<2>(sfw + C::kSfwCols * kt + 4 * i, scale_desc(s + C::kOffSf + C::kSfa + (i * E::kKt + kt) * 512));
          }
#pragma unroll
          for (int j = 0; j < E::kMma; ++j)
            mma_bs_w<2, F4>(d, smem_desc_k_sw128(s + j * 32), smem_desc_k_sw128(s + C::kA + j * 32),
                            idesc | idesc_sf(E::sf_of(j)), sfa + 4 * E::kt_of(j), sfw + C::kSfwCols * E::kt_of(j),
                            (ks > 0 || j > 0) ? 1u : 0u);
          mma_commit_pair_w(&empty[st]);
          if (++st == C::kStages) {
            st = 0;
            phase ^= 1u;
          }
        }
        if (ok) mma_commit_pair_w(&acc_full[buf]);
      }
      mma_commit_pair_w(mma_done);
    }
  } else {
    const int e = warp - 2, q = warp & 3;
    const int set = e >> 3;      // BN 256: the shared half of every tile or the other one; BN 128: even or odd tiles
    const int h = (e >> 2) & 1;  // which 64 columns of the 128
    constexpr int kEvery = BN == 256 ? 1 : 2;  // this warp's tiles among the pair's
    uint8_t* stg = smem + C::kOffStaging + e * C::kStaging;
    float* bias = reinterpret_cast<float*>(smem + C::kOffBias) + e * 64;
    const uint32_t lane_base = tmem + (static_cast<uint32_t>(q * 32) << 16);
    const uint32_t free_bars = cluster_map(smem_addr(acc_free), 0);
    constexpr int kCols = C::kRow / static_cast<int>(sizeof(T));  // columns of a staging row: 64, 32 or 16
    // the swizzle of 128-byte or 64-byte rows: 16-byte chunk j of row r is at chunk (j ^ swz(r))
    auto swz = [](int r) { return C::kRow == 128 ? (r & 7) : ((r >> 1) & 3); };
    // first tensor-memory column and first row and column of the output of this warp's part of tile t (the local-th)
    auto part_of = [&](int t, int local, int& col, int& row0, int& col0) {
      int mt, nt;
      tile_at(t, mt, nt);
      row0 = mt * 256 + static_cast<int>(rank) * 128 + q * 32;
      if (BN == 256) {
        col = (set == 0 ? 128 : (local & 1) ? 256 : 0) + h * 64;
        col0 = nt * 256 + col - (local & 1) * 128;
      } else {
        col = local % NA * 128 + h * 64;
        col0 = nt * 128 + h * 64;
      }
    };
    auto load_bias = [&](int col0, float& b0, float& b1) {  // columns 2 lane and 2 lane + 1
      const int n = col0 + 2 * lane;
      b0 = a.bias && n < a.N ? __ldg(a.bias + n) : 0.f;
      b1 = a.bias && n + 1 < a.N ? __ldg(a.bias + n + 1) : 0.f;
    };
    int local = BN == 256 ? 0 : set, col = 0, row0 = 0, col0 = 0;
    int t = pair + local * a.n_pairs;
    float b0 = 0.f, b1 = 0.f;
    if (t < total) {
      part_of(t, local, col, row0, col0);
      load_bias(col0, b0, b1);
    }
    for (; t < total; t += kEvery * a.n_pairs, local += kEvery) {
      __syncwarp();
      *reinterpret_cast<float2*>(bias + 2 * lane) = make_float2(b0, b1);
      __syncwarp();
      const int tcol = col, r0 = row0, c0 = col0;
      if (t + kEvery * a.n_pairs < total) {  // the next tile's bias comes while this tile is worked on
        part_of(t + kEvery * a.n_pairs, local + kEvery, col, row0, col0);
        load_bias(col0, b0, b1);
      }
      if (!mbar_wait_warp(&acc_full[local % NA], static_cast<uint32_t>(local / NA) & 1u, abort_flag)) break;
      tc_fence_after();
      // BN 256: both chunks at once, for the next tile's MMAs wait on the shared half. BN 128: one after the other, which
      // leaves registers for more of the activation at a time.
      constexpr bool kBoth = BN == 256;
      uint32_t r[kBoth ? 2 : 1][32];
      auto release = [&] {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) arrive_leader(free_bars + (BN == 256 && set == 0 ? NA : local % NA) * 8);
      };
      if (kBoth) {
        tmem_ld_32x32b_x32(lane_base + tcol, r[0]);
        tmem_ld_32x32b_x32(lane_base + tcol + 32, r[kBoth ? 1 : 0]);
        tmem_ld_wait_regs(r[0]);
        tmem_ld_wait_regs(r[kBoth ? 1 : 0]);
        release();
      }
      if (r0 >= a.M || c0 >= a.N) {
        if (!kBoth) release();
        continue;
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const uint32_t(&rc)[32] = r[kBoth ? c : 0];
        if (!kBoth) {
          tmem_ld_32x32b_x32(lane_base + tcol + c * 32, r[0]);
          tmem_ld_wait_regs(r[0]);
          if (c == 1) release();
        }
        float v[32];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float4 b = reinterpret_cast<const float4*>(bias)[c * 8 + j];
          v[4 * j] = __uint_as_float(rc[4 * j]) + b.x;
          v[4 * j + 1] = __uint_as_float(rc[4 * j + 1]) + b.y;
          v[4 * j + 2] = __uint_as_float(rc[4 * j + 2]) + b.z;
          v[4 * j + 3] = __uint_as_float(rc[4 * j + 3]) + b.w;
        }
        apply_act(v, a.act);
        constexpr int kPart = kCols < 32 ? kCols : 32;  // columns of this chunk in one store
#pragma unroll
        for (int part = 0; part < 32 / kPart; ++part) {
          const float* w = v + part * kPart;
          if (kCols <= 32 || c == 0) {
            if (lane == 0) bulk_wait_read<0>();  // the last store has left the tile
            __syncwarp();
          }
          constexpr int kChunks = kPart * static_cast<int>(sizeof(T)) / 16;
          const int first = kCols <= 32 ? 0 : c * kChunks;
#pragma unroll
          for (int j = 0; j < kChunks; ++j) {
            uint4 u;
            if constexpr (sizeof(T) == 4)
              u = make_uint4(__float_as_uint(w[4 * j]), __float_as_uint(w[4 * j + 1]), __float_as_uint(w[4 * j + 2]),
                             __float_as_uint(w[4 * j + 3]));
            else
              u = make_uint4(pack2<T>(w[8 * j], w[8 * j + 1]), pack2<T>(w[8 * j + 2], w[8 * j + 3]),
                             pack2<T>(w[8 * j + 4], w[8 * j + 5]), pack2<T>(w[8 * j + 6], w[8 * j + 7]));
            *reinterpret_cast<uint4*>(stg + lane * C::kRow + (((first + j) ^ swz(lane)) << 4)) = u;
          }
          if (kCols > 32 && c == 0) continue;  // the other chunk fills the row
          const int pc = c0 + (kCols > 32 ? 0 : c * 32 + part * kPart);
          if (a.tma_out) {
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0 && pc < a.N) {
              tma_store_2d(&map_out, stg, pc, r0);
              bulk_commit();
            }
          } else {
            __syncwarp();
            T* out = static_cast<T*>(a.out);
            const int rows = static_cast<int>(min(int64_t(32), a.M - r0));
#pragma unroll 8
            for (int i = lane; i < rows * kCols; i += 32) {
              const int rr = i / kCols, cc = i % kCols, byte = cc * static_cast<int>(sizeof(T));
              if (pc + cc < a.N)
                out[static_cast<int64_t>(r0 + rr) * a.N + pc + cc] =
                    *reinterpret_cast<const T*>(stg + rr * C::kRow + (((byte >> 4) ^ swz(rr)) << 4) + (byte & 15));
            }
            __syncwarp();
          }
        }
      }
    }
    if (lane == 0) bulk_wait<0>();  // the stores have left shared memory and are written
  }
  tc_fence_before();
  __syncthreads();
  // Also after an abort, what was issued completes before its memory is given back. The wait comes after the CTA's other roles
  // have ended, whose waits cover a tile each: begun at the start, it would put its limit on the whole product. After an abort
  // loads may be in flight that no MMA waited for, too. They land within microseconds, and their barrier may be the peer's, so
  // this CTA gives them ten milliseconds before it leaves.
  if (warp == 1) {
    volatile int never = 0;
    if (!mbar_wait_warp(mma_done, 0, &never)) *abort_flag = 1;
    if (*abort_flag) {
      const uint64_t t0 = globaltimer_ns();
      while (globaltimer_ns() - t0 < 10000000ull) {}
    }
    __syncwarp();
  }
  cluster_sync();  // neither CTA leaves while the other's arrivals, copies or MMAs may still reach it
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, 512);
  }
  if (threadIdx.x == 0 && *abort_flag && a.dev_status) atomicExch(a.dev_status, KO_ERR_DEVICE_TIMEOUT);
}

// ---------------------------------------------------------------------------------------------------------
// slice_kernel: few rows of A. The weight's rows take the MMA's 128-row side and A's rows (BN of them) its narrow side, so
// the product comes out transposed: a thread owns one output column and a warp writes 32 neighbours of a row at a time, for
// any N. The CTAs of a cluster share a tile and take a slice of K each; their partial sums meet in shared memory and are
// added in rank order through distributed shared memory, so results repeat bit for bit.
// With XT other than void the rows of A come as XT values, at most kFuseRows of them, and four groups of two more warps
// quantise them to mxfp4 on the way into shared memory, each every fourth stage and a block of 32 to a thread: for a handful
// of tokens that costs less than a launch of its own, and every CTA needs only its slice of them. (One group, even with the
// next stage's elements on their way, was the slowest part: 1 x 8192 x 8192 in 13.2 us, 10.8 with four.)
// ---------------------------------------------------------------------------------------------------------
constexpr int kSliceThreads = 128;   // without the quantising warps
constexpr int kFuseGroups = 4, kFuseThreads = 64 + 64 * kFuseGroups;
constexpr int kFuseRows = KO_MXFP4_FUSED_ROWS;

struct SliceArgs {
  const float* bias;
  void* out;
  int* dev_status;
  int64_t M, N;
  int act, k_stages, n_tiles, slices;
  int vec_out;    // four neighbours of a row of out can be stored at once
  const void* x;  // unquantised rows [M][K], ldx elements apart (XT other than void)
  int64_t K, ldx;
  int x_vec;      // rows of x are whole groups of eight (groups_of_8)
};

// Adds the S partial sums of rows rank, rank + S, ... of a tile and stores them. A warp takes 8 / S rows at a time and a lane
// four columns of them: eight 128-bit reads through distributed shared memory on their way at once, added in rank order.
template <int S, typename T>
__device__ __forceinline__ void add_slices(const SliceArgs& a, float* part, int nt, int64_t m0, int cols, int rank) {
  constexpr int R = 8 / S;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t n = static_cast<int64_t>(nt) * 128 + lane * 4;
  uint32_t from[S];
#pragma unroll
  for (int s = 0; s < S; ++s) from[s] = cluster_map(smem_addr(part) + lane * 16, static_cast<uint32_t>(s));
  float bias[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) bias[i] = a.bias && n + i < a.N ? __ldg(a.bias + n + i) : 0.f;
  for (int j0 = rank + S * R * warp; j0 < cols; j0 += S * R * (kSliceThreads / 32)) {
    float4 p[R][S];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int s = 0; s < S; ++s) {
        p[r][s] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (j0 + r * S < cols) p[r][s] = cluster_load_f4(from[s] + (j0 + r * S) * 512);
      }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int j = j0 + r * S;
      if (j >= cols) break;
      float v[4] = {p[r][0].x, p[r][0].y, p[r][0].z, p[r][0].w};
#pragma unroll
      for (int s = 1; s < S; ++s) {
        v[0] += p[r][s].x;
        v[1] += p[r][s].y;
        v[2] += p[r][s].z;
        v[3] += p[r][s].w;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] += bias[i];
      apply_act(v, a.act);
      T* o = static_cast<T*>(a.out) + (m0 + j) * a.N + n;
      if (n + 4 <= a.N && a.vec_out) {
        if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(o) = make_float4(v[0], v[1], v[2], v[3]);
        else *reinterpret_cast<uint2*>(o) = make_uint2(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]));
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (n + i < a.N) o[i] = from_f<T>(v[i]);
      }
    }
  }
}

template <bool F4, int BN, typename T, typename XT>
__global__ void __launch_bounds__(std::is_void<XT>::value ? kSliceThreads : kFuseThreads)
    slice_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w,
                 const __grid_constant__ CUtensorMap map_sx, const __grid_constant__ CUtensorMap map_sw,
                 const SliceArgs a) {
  using C = SliceCfg<F4, BN>;
  using E = Elem<F4>;
  constexpr bool kFuse = !std::is_void<XT>::value;
  static_assert(!kFuse || (F4 && BN == kFuseRows), "fused quantisation is for mxfp4 and one tile of rows");
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::kOffBars);
  uint64_t* empty = full + C::kStages;
  uint64_t* acc_full = empty + C::kStages;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_full + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int S = a.slices;
  const int rank = static_cast<int>(blockIdx.x % S), tile = static_cast<int>(blockIdx.x / S);
  const int nt = tile % a.n_tiles, mt = tile / a.n_tiles;
  const int k0 = static_cast<int>(static_cast<int64_t>(a.k_stages) * rank / S);
  const int k1 = static_cast<int>(static_cast<int64_t>(a.k_stages) * (rank + 1) / S);
  const int64_t m0 = static_cast<int64_t>(mt) * BN;
  const int cols = static_cast<int>(min(int64_t(BN), a.M - m0));  // rows of A in this tile

  wait_for_previous_grid();
  auto load_stage = [&](int ks, int st) {
    uint8_t* s = smem + st * C::kStage;
    mbar_arrive_expect_tx(&full[st], kFuse ? Elem<F4>::kTxW + C::kSf : C::kTx);
    tma_load_2d(&map_w, &full[st], s, ks * 128, nt * 128);
    tma_load_2d(&map_sw, &full[st], s + C::kOffSf, ks * 64 * E::kKt, nt);
    if (!kFuse) {
      tma_load_2d(&map_x, &full[st], s + C::kW, ks * 128, static_cast<int32_t>(m0));
      tma_load_2d(&map_sx, &full[st], s + C::kOffSf + C::kSf, ks * 64 * E::kKt, static_cast<int32_t>(m0 / 128));
    }
  };
  const int ahead = min(C::kStages, k1 - k0);  // stages that are loaded before anything else is set up
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(&full[s], kFuse ? 3 : 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(acc_full, 1);
    *abort_flag = 0;
    fence_barrier_init();
    fence_proxy_async_smem();
    for (int i = 0; i < ahead; ++i) load_stage(k0 + i, i);
  }
  if (kFuse && warp >= 2) {  // the scale tiles of x hold kFuseRows rows; the others are zero for good
    for (int i = threadIdx.x - 64; i < C::kStages * static_cast<int>(C::kSf / 4); i += kFuseThreads - 64) {
      const int st = i / static_cast<int>(C::kSf / 4), w = i % static_cast<int>(C::kSf / 4);
      reinterpret_cast<uint32_t*>(smem + st * C::kStage + C::kOffSf + C::kSf)[w] = 0u;
    }
    fence_proxy_async_smem();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, C::kCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    if (lane == 0) {
      int st = ahead % C::kStages, issued = ahead;
      uint32_t phase = 0;  // of the MMAs that free a stage
      for (int ks = k0 + ahead; ks < k1; ++ks) {
        if (!mbar_wait(&empty[st], phase, abort_flag)) break;
        load_stage(ks, st);
        ++issued;
        if (++st == C::kStages) {
          st = 0;
          phase ^= 1u;
        }
      }
      // every load has landed before the CTA leaves: the last use of each stage, the only one that may be in flight
      volatile int never = 0;
      for (int s = 0; s < C::kStages && s < issued; ++s) {
        const int last = (issued - 1 - s) / C::kStages;
        if (!mbar_wait(&full[s], static_cast<uint32_t>(last) & 1u, &never)) *abort_flag = 1;
      }
    }
  } else if (warp == 1) {
    constexpr uint32_t idesc = idesc_bs(E::kTypeW, E::kTypeA, 128, BN);
    const uint32_t sb = smem_addr(smem);
    int st = 0;
    uint32_t phase = 0;
    for (int ks = k0; ks < k1; ++ks) {
      if (!mbar_wait_warp(&full[st], phase, abort_flag)) break;
      tc_fence_after();
      const uint32_t s = sb + st * C::kStage;
      const uint32_t sfw = tmem + C::kAccCols + st * C::kSfCols, sfx = sfw + 4 * E::kKt;
#pragma unroll
      for (int kt = 0; kt < E::kKt; ++kt) {
        cp_scales_w<1>(sfw + 4 * kt, scale_desc(s + C::kOffSf + kt * 512));
        cp_scales_w<1>(sfx + 4 * kt, scale_desc(s + C::kOffSf + C::kSf + kt * 512));
      }
#pragma unroll
      for (int j = 0; j < E::kMma; ++j)
        mma_bs_w<1, F4>(tmem, smem_desc_k_sw128(s + j * 32), smem_desc_k_sw128(s + C::kW + j * 32),
                        idesc | idesc_sf(E::sf_of(j)), sfw + 4 * E::kt_of(j), sfx + 4 * E::kt_of(j),
                        (ks > k0 || j > 0) ? 1u : 0u);
      mma_commit_w(&empty[st]);
      if (++st == C::kStages) {
        st = 0;
        phase ^= 1u;
      }
    }
    mma_commit_w(acc_full);
  } else if constexpr (kFuse) {
    // Two blocks of a stage per thread: block b of rows r and r + 8. A block's codes are one 16-byte chunk of the row.
    const int b = threadIdx.x & 7, r = (threadIdx.x >> 3) & 7;
    for (int ks = k0 + ((warp - 2) >> 1); ks < k1; ks += kFuseGroups) {
      Raw8<XT> raw[2][4];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int64_t k = static_cast<int64_t>(ks) * E::kStageK + b * 32;
        const XT* p = static_cast<const XT*>(a.x) + (r + 8 * i) * a.ldx + k;
        const int left = r + 8 * i < cols ? static_cast<int>(a.K - k) : 0;
        if (a.x_vec) load_block<XT, true>(p, left, raw[i]);
        else load_block<XT, false>(p, left, raw[i]);
      }
      uint32_t code[2][4], byte[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) byte[i] = quantize_block<XT, KO_MXFP4, 1>(raw[i], code[i]);
      const int st = (ks - k0) % C::kStages;
      const uint32_t phase = static_cast<uint32_t>((ks - k0) / C::kStages) & 1u;
      if (!mbar_wait_warp(&empty[st], phase ^ 1u, abort_flag)) break;
      uint8_t* s = smem + st * C::kStage;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int row = r + 8 * i;
        *reinterpret_cast<uint4*>(s + C::kW + row * 128 + ((b ^ (row & 7)) << 4)) =
            make_uint4(code[i][0], code[i][1], code[i][2], code[i][3]);
        s[C::kOffSf + C::kSf + (b >> 2) * 512 + row * 16 + (b & 3)] = static_cast<uint8_t>(byte[i]);
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&full[st]);
    }
  }
  __syncwarp();
  volatile int never = 0;  // also after an abort: what was issued completes before its memory is given back
  if (!mbar_wait_warp(acc_full, 0, &never)) *abort_flag = 1;
  tc_fence_after();

  const int64_t n = static_cast<int64_t>(nt) * 128 + threadIdx.x;
  const float bias = a.bias && n < a.N ? __ldg(a.bias + n) : 0.f;
  T* out = static_cast<T*>(a.out) + m0 * a.N + n;
  float* part = reinterpret_cast<float*>(smem);  // [BN][128]: every load has been read by its MMAs
  const uint32_t lane_base = tmem + (static_cast<uint32_t>(warp * 32) << 16);
  const bool epilogue = !kFuse || warp < kSliceThreads / 32;
#pragma unroll
  for (int c = 0; c < (BN + 31) / 32; ++c) {
    if (c * 32 >= cols || !epilogue) break;
    uint32_t r[32];
    tmem_ld_32x32b_x32(lane_base + c * 32, r);
    tmem_ld_wait_regs(r);
    if (S > 1) {
#pragma unroll
      for (int j = 0; j < 32; ++j)
        if (c * 32 + j < cols) part[(c * 32 + j) * 128 + threadIdx.x] = __uint_as_float(r[j]);
      continue;
    }
    float v[32];
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(r[j]) + bias;
    apply_act(v, a.act);
    if (n < a.N) {
#pragma unroll
      for (int j = 0; j < 32; ++j)
        if (c * 32 + j < cols) out[(c * 32 + j) * a.N] = from_f<T>(v[j]);
    }
  }
  tc_fence_before();
  if (S > 1) {
    cluster_sync();
    if (epilogue) {
      if (S == 2) add_slices<2, T>(a, part, nt, m0, cols, rank);
      else if (S == 4) add_slices<4, T>(a, part, nt, m0, cols, rank);
      else add_slices<8, T>(a, part, nt, m0, cols, rank);
    }
    cluster_sync();  // no CTA leaves while another reads its sums
  } else {
    __syncthreads();
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, C::kCols);
  }
  if (threadIdx.x == 0 && *abort_flag && a.dev_status) atomicExch(a.dev_status, KO_ERR_DEVICE_TIMEOUT);
}

// ---- host ---------------------------------------------------------------------------------------------------

int encode_2d(CUtensorMap* map, CUtensorMapDataType type, const void* base, uint64_t cols, uint64_t rows,
              uint64_t pitch_bytes, uint32_t box_cols, uint32_t box_rows, CUtensorMapSwizzle swizzle, const char* what) {
  ko::EncodeTiledFn enc = ko::encode_tiled();
  if (!enc) return ko::fail(KO_ERR_UNSUPPORTED, "cuTensorMapEncodeTiled is not available from the driver");
  cuuint64_t dims[2] = {cols, rows}, strides[1] = {pitch_bytes};
  cuuint32_t box[2] = {box_cols, box_rows}, estr[2] = {1, 1};
  const CUresult r = enc(map, type, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return ko::fail(KO_ERR_INVALID_ARGUMENT,
                    std::string(what) + ": cuTensorMapEncodeTiled failed (CUresult " + std::to_string(r) + ")");
  return KO_OK;
}
// Boxes of 128 shared-memory bytes x box_rows rows; `spread`: 4-bit codes to one per byte.
int encode_codes(CUtensorMap* map, const void* codes, int fmt, bool spread, int64_t rows, int64_t Kp, uint32_t box_rows,
                 const char* what) {
  const uint64_t pitch = static_cast<uint64_t>(fmt == KO_MXFP4 ? Kp / 2 : Kp);
  if (spread)
    return encode_2d(map, CU_TENSOR_MAP_DATA_TYPE_16U4_ALIGN16B, codes, Kp, rows, pitch, 128, box_rows,
                     CU_TENSOR_MAP_SWIZZLE_128B, what);
  return encode_2d(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, codes, pitch, rows, pitch, 128, box_rows,
                   CU_TENSOR_MAP_SWIZZLE_128B, what);
}
// Scale tiles as rows of 64 8-byte words per tile; boxes of kt tiles along K x row_tiles.
int encode_scales(CUtensorMap* map, const void* scales, int64_t rows, int64_t Kp, int kt, uint32_t row_tiles,
                  const char* what) {
  const uint64_t words = static_cast<uint64_t>(Kp / 128) * 64;
  return encode_2d(map, CU_TENSOR_MAP_DATA_TYPE_UINT64, scales, words, static_cast<uint64_t>((rows + 127) / 128),
                   words * 8, 64u * kt, row_tiles, CU_TENSOR_MAP_SWIZZLE_NONE, what);
}

struct Call {
  const void *ac, *as, *wc, *ws;
  const float* bias;
  int64_t M, K, N, Kp;
  int act;
  void* out;
  int* dev_status;
  cudaStream_t stream;
  const ko::DeviceInfo* info;
  const void* x;  // unquantised A (fused form)
  int64_t ldx;
  // Launched straight behind the kernel that quantises A: sets itself up while that one finishes (25664 x 384 x 1536 with
  // its quantisation 57.8 -> 55.7 us, 301 x 1000 x 517 on the device 9.9 -> 8.9).
  bool behind;
};

// The opt-in to more than 48 KB of shared memory, once per kernel and device.
template <typename Kernel>
int allow_smem(Kernel kernel, std::atomic<bool>* done, int dev, uint32_t bytes) {
  if (done[dev].load(std::memory_order_relaxed)) return KO_OK;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
  if (e != cudaSuccess) return ko::fail(static_cast<int>(e), "ko_linear_mxfp4: shared memory");
  done[dev].store(true, std::memory_order_relaxed);
  return KO_OK;
}
constexpr int kMaxDevices = 64;
int current_device() {  // device_or_fail has accepted it, so it is below kMaxDevices
  int dev = 0;
  return cudaGetDevice(&dev) == cudaSuccess && dev >= 0 && dev < kMaxDevices ? dev : 0;
}

cudaLaunchConfig_t cluster_config(cudaLaunchAttribute (&attr)[2], unsigned cluster, unsigned blocks, unsigned threads,
                                  size_t smem, const Call& c) {
  cudaLaunchConfig_t cfg = {};
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.gridDim = dim3(blocks);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.stream = c.stream;
  cfg.attrs = attr;
  cfg.numAttrs = c.behind ? 2 : 1;
  return cfg;
}

template <bool F4, int BN, typename T>
int launch_pair(const Call& c) {
  using C = PairCfg<F4, BN>;
  using E = Elem<F4>;
  constexpr const char* who = "ko_linear_mxfp4";
  const int64_t mt = (c.M + 255) / 256, nt = (c.N + BN - 1) / BN;
  CUtensorMap ma, mw, msa, msw, mo;
  const int64_t es = static_cast<int64_t>(sizeof(T));
  const bool tma_out = ko::aligned16(c.out) && c.N * es % 16 == 0;
  int rc = encode_codes(&ma, c.ac, F4 ? KO_MXFP4 : KO_MXFP8, false, c.M, c.Kp, 128, who);
  if (!rc) rc = encode_codes(&mw, c.wc, KO_MXFP4, !F4, c.N, c.Kp, BN / 2, who);
  if (!rc) rc = encode_scales(&msa, c.as, c.M, c.Kp, E::kKt, 1, who);
  if (!rc) rc = encode_scales(&msw, c.ws, c.N, c.Kp, E::kKt, BN / 128, who);
  mo = ma;  // not used without tma_out
  if (!rc && tma_out)
    rc = encode_2d(&mo, es == 4 ? CU_TENSOR_MAP_DATA_TYPE_UINT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16, c.out, c.N, c.M,
                   c.N * es, static_cast<uint32_t>(C::kRow / es), 32,
                   C::kRow == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, who);
  if (rc) return rc;
  PairArgs a{};
  a.bias = c.bias;
  a.out = c.out;
  a.dev_status = c.dev_status;
  a.M = c.M;
  a.N = c.N;
  a.act = c.act;
  a.k_stages = static_cast<int>((c.Kp + E::kStageK - 1) / E::kStageK);
  a.m_tiles = static_cast<int>(mt);
  a.n_tiles = static_cast<int>(nt);
  a.tma_out = tma_out ? 1 : 0;
  auto kernel = pair_kernel<F4, BN, T>;
  static std::atomic<bool> allowed[kMaxDevices];
  static std::atomic<int> resident[kMaxDevices];  // CTA pairs that the device holds at once, found once per device
  const int dev = current_device();
  rc = allow_smem(kernel, allowed, dev, C::kSmem);
  if (rc) return rc;
  cudaLaunchAttribute attr[2];
  cudaLaunchConfig_t cfg =
      cluster_config(attr, 2, 2 * static_cast<unsigned>(c.info->sm_count / 2), kPairThreads, C::kSmem, c);
  int pairs = resident[dev].load(std::memory_order_relaxed);
  if (pairs <= 0) {
    const cudaError_t e = cudaOccupancyMaxActiveClusters(&pairs, kernel, &cfg);
    if (e != cudaSuccess) return ko::fail(static_cast<int>(e), std::string(who) + ": occupancy");
    pairs = std::max(pairs, 1);
    resident[dev].store(pairs, std::memory_order_relaxed);
  }
  a.n_pairs = static_cast<int>(std::min<int64_t>(mt * nt, pairs));
  cfg.gridDim = dim3(2 * static_cast<unsigned>(a.n_pairs));
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, ma, mw, msa, msw, mo, a);
  if (e != cudaSuccess) return ko::fail(static_cast<int>(e), std::string(who) + ": launch failed");
  return ko::check_launch(who);
}

template <bool F4, int BN, typename T, typename XT = void>
int launch_slice(const Call& c) {
  constexpr bool kFuse = !std::is_void<XT>::value;
  using C = SliceCfg<F4, BN>;
  using E = Elem<F4>;
  constexpr const char* who = "ko_linear_mxfp4";
  const int64_t mt = (c.M + BN - 1) / BN, nt = (c.N + 127) / 128;
  CUtensorMap mx, mw, msx, msw;
  int rc = encode_codes(&mw, c.wc, KO_MXFP4, !F4, c.N, c.Kp, 128, who);
  if (!rc) rc = encode_scales(&msw, c.ws, c.N, c.Kp, E::kKt, 1, who);
  if (kFuse) {
    mx = mw;  // not used
    msx = msw;
  } else {
    if (!rc) rc = encode_codes(&mx, c.ac, F4 ? KO_MXFP4 : KO_MXFP8, false, c.M, c.Kp, BN, who);
    if (!rc) rc = encode_scales(&msx, c.as, c.M, c.Kp, E::kKt, 1, who);
  }
  if (rc) return rc;
  SliceArgs a{};
  if constexpr (kFuse) {
    a.x = c.x;
    a.K = c.K;
    a.ldx = c.ldx;
    a.x_vec = reinterpret_cast<uintptr_t>(c.x) % (8 * sizeof(XT)) == 0 && c.ldx % 8 == 0 && c.K % 8 == 0;
  }
  a.bias = c.bias;
  a.out = c.out;
  a.dev_status = c.dev_status;
  a.M = c.M;
  a.N = c.N;
  a.act = c.act;
  a.k_stages = static_cast<int>((c.Kp + E::kStageK - 1) / E::kStageK);
  a.n_tiles = static_cast<int>(nt);
  // Slices of K: as many as two CTAs on every SM hold, in clusters of eight only where one on every SM will do (1 x 4096 x
  // 4096 in 7.3 us with eight, 6.7 with four; 1 x 8192 x 1024 in 6.7 and 9.0).
  int slices = 1;
  while (slices < 8 && mt * nt * slices * 2 <= (slices == 4 ? 1 : 2) * c.info->sm_count && slices * 2 <= a.k_stages)
    slices *= 2;
  a.slices = slices;
  a.vec_out = c.N % 4 == 0 && reinterpret_cast<uintptr_t>(c.out) % (4 * sizeof(T)) == 0;
  auto kernel = slice_kernel<F4, BN, T, XT>;
  static std::atomic<bool> allowed[kMaxDevices];
  rc = allow_smem(kernel, allowed, current_device(), C::kSmem);
  if (rc) return rc;
  cudaLaunchAttribute attr[2];
  cudaLaunchConfig_t cfg = cluster_config(attr, slices, static_cast<unsigned>(mt * nt * slices),
                                          kFuse ? kFuseThreads : kSliceThreads, C::kSmem,
                                          c);
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, mx, mw, msx, msw, a);
  if (e != cudaSuccess) return ko::fail(static_cast<int>(e), std::string(who) + ": launch failed");
  return ko::check_launch(who);
}

// Which kernel, by the numbers of 256 x 128 tiles and of pipeline stages along K (mxfp4, bf16 outputs, us on B200):
//   up to 64 rows, the slices: 48 x 8192 x 8192 in 9.9 against 14.8 with pairs.
//   Up to 128 rows read the weight once, and a pair's tile would be half empty: the slices too, from 16 stages on (128 x 4096 x
//   4096 in 8.8 against 10.2, 128 x 8192 x 20480 in 19.7 against 29.9; 128 x 2048 x 4096, eight stages, in 8.2 against 7.8).
//   More rows, but no more tiles than stages, for the pairs would leave SMs idle behind a long K: the slices while a device
//   with a CTA per 128 x 128 tile has SMs left to cut K for (300 x 4096 x 512 in 7.6 against 9.8; with more tiles than stages
//   the pairs, 1200 x 4096 x 512 in 10.0 against 10.2, 1200 x 1024 x 1024 in 6.8 against 8.0). In mxfp8, 144 such tiles:
//   1024 x 16384 x 2304 in 33 against 43, and 160, a second round of whole K: 1024 x 16384 x 2560 in 49 against 44, 768 x
//   28672 x 8192 in 186 against 146.
//   Pairs with 256 x 128 tiles while these fill one round of the SMs (300 x 4096 x 4096 in 10.0 against 11.6), or where K is so
//   short that the epilogue counts, over five shapes from 16384 x 1024 to 4096 x 8192 outputs. With GELU up to four stages: 1 to
//   12 % faster than 256 x 256 (25664 x 1024 x 1536 in 45.6 against 49.2; with five 2 % slower to 6 % faster). Without it up to
//   two: with 16-bit outputs 6 to 17 % faster at one stage (8192 x 256 x 4096 in 17.9 against 20.5), 4 % faster to 2 % slower at
//   two and up to 11 % slower at three; with fp32 outputs, bound by their stores, 5 % faster to 9 % slower at one and two (4096 x
//   512 x 8192 in 31.2 against 28.2), but 16 to 18 % faster where rows are not on 16 bytes (12000 x 512 x 2999 in 71 against 84).
//   Else 256 x 256, with less to load for a product (25664 x 2048 x 1536 with GELU in 56 against 65, 4096 x 8192 x 8192 in 99
//   against 145).
template <bool F4, typename T>
int launch(const Call& c) {
  const int64_t tiles = ((c.M + 255) / 256) * ((c.N + 127) / 128);
  const int64_t stages = (c.Kp + Elem<F4>::kStageK - 1) / Elem<F4>::kStageK;
  if (c.M <= 16) return launch_slice<F4, 16, T>(c);
  if (c.M <= 32) return launch_slice<F4, 32, T>(c);
  if (c.M <= 64) return launch_slice<F4, 64, T>(c);
  if (c.M <= 128 && stages >= 16) return launch_slice<F4, 128, T>(c);
  if (tiles <= stages && (c.M + 127) / 128 * ((c.N + 127) / 128) <= c.info->sm_count) return launch_slice<F4, 128, T>(c);
  if (tiles <= c.info->sm_count / 2 || stages <= (c.act == KO_ACT_GELU ? 4 : 2)) return launch_pair<F4, 128, T>(c);
  return launch_pair<F4, 256, T>(c);
}

template <typename T>
int launch_fused(const Call& c, int x_dtype) {
  if (x_dtype == KO_F32) return launch_slice<true, kFuseRows, T, float>(c);
  if (x_dtype == KO_BF16) return launch_slice<true, kFuseRows, T, __nv_bfloat16>(c);
  return launch_slice<true, kFuseRows, T, __half>(c);
}

int check_linear(const char* name, int64_t M, int64_t K, int64_t N, int act, const void* w_codes, const void* w_scales,
                 const float* bias, const void* out, int out_dtype) {
  auto bad = [&](const char* what) { return ko::fail(KO_ERR_INVALID_ARGUMENT, std::string(name) + ": " + what); };
  if (M < 0 || M > kMaxRows || K < 1 || K > kMaxK || N < 1 || N > kMaxRows)
    return bad("need 0 <= M <= 2^31, 1 <= K <= 2^24 and 1 <= N <= 2^31");
  // Tiles are counted in 32 bits, with room for a band of eight or a cluster of eight slices. Checked here, before anything
  // is launched; it holds M * N to 2^42.
  if (((M + 255) / 256) * ((N + 127) / 128) > INT32_MAX / 16) return bad("too many output tiles");
  if (!dtype_ok(out_dtype)) return bad("unknown output type");
  if (act != KO_ACT_NONE && act != KO_ACT_GELU && act != KO_ACT_RELU)
    return bad("act must be KO_ACT_NONE, KO_ACT_GELU or KO_ACT_RELU");
  if (M == 0) return KO_OK;
  if (!w_codes || !w_scales || !out) return bad("null pointer");
  if (reinterpret_cast<uintptr_t>(w_codes) % 32 != 0 || !ko::aligned16(w_scales))
    return bad("the weight's codes must be 32-byte aligned, its scales 16");
  if (reinterpret_cast<uintptr_t>(out) % static_cast<uintptr_t>(dtype_size(out_dtype)) != 0 ||
      reinterpret_cast<uintptr_t>(bias) % 4 != 0)
    return bad("out and bias must be aligned to their elements");
  return KO_OK;
}

// The weight and the bias as what an output may not overlap.
struct Operands {
  Range codes, scales, bias;
};
Operands operands(const void* w_codes, const void* w_scales, const float* bias, int64_t K, int64_t N) {
  return {{w_codes, ko_mx_codes_bytes(N, K, KO_MXFP4)}, {w_scales, ko_mx_scales_bytes(N, K)}, {bias, 4 * N}};
}

// ko_linear_mxfp4 after the checks of its operands.
int product(Call c, int a_fmt, int out_dtype, const char* name) {
  const int rc = ko::device_or_fail(&c.info, name);
  if (rc) return rc;
  const bool f4 = a_fmt == KO_MXFP4;
  if (out_dtype == KO_F32) return f4 ? launch<true, float>(c) : launch<false, float>(c);
  if (out_dtype == KO_BF16) return f4 ? launch<true, __nv_bfloat16>(c) : launch<false, __nv_bfloat16>(c);
  return f4 ? launch<true, __half>(c) : launch<false, __half>(c);
}

}  // namespace

extern "C" int ko_linear_mxfp4(const void* a_codes, const void* a_scales, int a_fmt, const void* w_codes,
                               const void* w_scales, const float* bias, int64_t M, int64_t K, int64_t N, int act,
                               void* out, int out_dtype, int* dev_status, ko_stream_t stream) {
  const char* name = "ko_linear_mxfp4";
  const int rc = check_linear(name, M, K, N, act, w_codes, w_scales, bias, out, out_dtype);
  if (rc) return rc;
  if (!fmt_ok(a_fmt)) return ko::fail(KO_ERR_INVALID_ARGUMENT, "ko_linear_mxfp4: unknown format");
  if (M == 0) return KO_OK;
  if (!a_codes || !a_scales || !ko::aligned16(a_codes) || !ko::aligned16(a_scales))
    return ko::fail(KO_ERR_INVALID_ARGUMENT, "ko_linear_mxfp4: codes and scales must be given, 16-byte aligned");
  const Operands w = operands(w_codes, w_scales, bias, K, N);
  if (meets({out, M * N * dtype_size(out_dtype)}, {{a_codes, ko_mx_codes_bytes(M, K, a_fmt)},
                                                  {a_scales, ko_mx_scales_bytes(M, K)}, w.codes, w.scales, w.bias}))
    return ko::fail(KO_ERR_INVALID_ARGUMENT, "ko_linear_mxfp4: out overlaps an operand");
  return product(Call{a_codes, a_scales, w_codes, w_scales, bias, M, K, N, padded_k(K), act, out, dev_status,
                      reinterpret_cast<cudaStream_t>(stream), nullptr, nullptr, 0, false},
                 a_fmt, out_dtype, name);
}

extern "C" int64_t ko_linear_quantize_mxfp4_workspace_bytes(int64_t M, int64_t K) {
  const int64_t codes = ko_mx_codes_bytes(M, K, KO_MXFP4), scales = ko_mx_scales_bytes(M, K);
  if (codes < 0 || scales < 0) return -1;
  return M <= kFuseRows ? 0 : (codes + 15) / 16 * 16 + scales;
}

extern "C" int ko_linear_quantize_mxfp4(const void* x, int x_dtype, int64_t ldx, const void* w_codes,
                                        const void* w_scales, const float* bias, int64_t M, int64_t K, int64_t N,
                                        int act, void* out, int out_dtype, void* workspace, int64_t workspace_bytes,
                                        int* dev_status, ko_stream_t stream) {
  const char* name = "ko_linear_quantize_mxfp4";
  int rc = check_linear(name, M, K, N, act, w_codes, w_scales, bias, out, out_dtype);
  if (rc) return rc;
  auto bad = [&](const char* what) { return ko::fail(KO_ERR_INVALID_ARGUMENT, std::string(name) + ": " + what); };
  if (!dtype_ok(x_dtype)) return bad("unknown element type");
  if (ldx < K) return bad("ldx must be at least K");
  if (!extent_ok(M, ldx)) return bad("the rows' pitch spans more than 2^46 elements");
  if (M == 0) return KO_OK;
  if (!x || reinterpret_cast<uintptr_t>(x) % static_cast<uintptr_t>(dtype_size(x_dtype)) != 0)
    return bad("x must be given, aligned to its elements");
  const Operands w = operands(w_codes, w_scales, bias, K, N);
  const Range in = span_of(x, M, ldx, K, dtype_size(x_dtype)), to = {out, M * N * dtype_size(out_dtype)};
  if (meets(to, {in, w.codes, w.scales, w.bias})) return bad("out overlaps x, the weight or the bias");
  if (M > kFuseRows) {
    if (!workspace || !ko::aligned16(workspace) || workspace_bytes < ko_linear_quantize_mxfp4_workspace_bytes(M, K))
      return bad("the workspace must be 16-byte aligned and hold ko_linear_quantize_mxfp4_workspace_bytes(M, K) bytes");
    if (meets({workspace, ko_linear_quantize_mxfp4_workspace_bytes(M, K)}, {in, to, w.codes, w.scales, w.bias}))
      return bad("the workspace overlaps x, out, the weight or the bias");
    uint8_t* codes = static_cast<uint8_t*>(workspace);
    uint8_t* scales = codes + (ko_mx_codes_bytes(M, K, KO_MXFP4) + 15) / 16 * 16;
    rc = ko_quantize_mx(x, x_dtype, M, K, ldx, KO_MXFP4, codes, scales, stream);
    if (rc) return rc;
    return product(Call{codes, scales, w_codes, w_scales, bias, M, K, N, padded_k(K), act, out, dev_status,
                        reinterpret_cast<cudaStream_t>(stream), nullptr, nullptr, 0, true},
                   KO_MXFP4, out_dtype, name);
  }
  Call c{nullptr, nullptr, w_codes, w_scales, bias, M, K, N, padded_k(K), act, out, dev_status,
         reinterpret_cast<cudaStream_t>(stream), nullptr, x, ldx, false};
  rc = ko::device_or_fail(&c.info, name);
  if (rc) return rc;
  if (out_dtype == KO_F32) return launch_fused<float>(c, x_dtype);
  if (out_dtype == KO_BF16) return launch_fused<__nv_bfloat16>(c, x_dtype);
  return launch_fused<__half>(c, x_dtype);
}
