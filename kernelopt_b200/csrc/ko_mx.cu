// Microscaled quantisation, its inverse, the 4-bit weight layout, and the residual + root-mean-square norm whose output
// can be microscaled in the same pass. Formats and layout: ko_mx.cuh.
//
// All of these read and write each byte once; HBM bounds them where the instructions per element are kept few.
#include <cmath>
#include <string>

#include "ko_mx.cuh"

namespace {

using namespace komx;

constexpr int kThreads = 256;

// ---------------------------------------------------------------------------------------------------------
// Quantisation: L lanes take a block of 32 elements. L 1 for 16-bit rows that are whole groups of eight: a block's scale is
// worked out once and without shuffles (8192 x 8192 bf16 in 26.8 us, 6.3 TB/s; with four lanes to a block 115 instructions
// for eight elements, bound by their issue, 36.7 us). L 2 for such fp32 rows, 64 bytes to a lane (25600 x 1536 in 26.7 us,
// 6.7 TB/s; 30.2 with L 1 or 4). L 4 for rows that are read element by element, from nearer addresses (1203 x 1001 in
// 2.7 us, 6.1 with L 1). Items run over the blocks of a row, then rows; the rows that fill the last tile of 128 are
// included (scale 0, no codes).
// ---------------------------------------------------------------------------------------------------------
template <typename T, int FMT, bool VEC, int L>
__global__ void __launch_bounds__(kThreads) quantize_kernel(const T* __restrict__ x, int64_t rows, int64_t K,
                                                            int64_t ldx, int64_t items, uint32_t kblocks,
                                                            int64_t code_pitch, uint8_t* __restrict__ codes,
                                                            uint8_t* __restrict__ scales) {
  let_next_grid_start();  // the product behind it sets itself up meanwhile (ko_linear_quantize_mxfp4)
  // items: a multiple of 512 blocks, so every warp is whole, in range or not, and the lanes of a block stay together
  const int64_t item = static_cast<int64_t>(blockIdx.x) * (kThreads / L) + threadIdx.x / L;
  if (item >= items) return;
  const int part = threadIdx.x % L;
  const int64_t row = items <= 0xffffffffll ? static_cast<uint32_t>(item) / kblocks : item / kblocks;
  const uint32_t kb = static_cast<uint32_t>(item - row * kblocks);
  uint8_t* scale = scales + scale_word_offset(row, kb >> 2, kblocks >> 2) + (kb & 3);
  const bool real = row < rows;
  constexpr int kWords = (FMT == KO_MXFP4 ? 4 : 8) / L;
  uint32_t c[kWords];
  const int64_t k = static_cast<int64_t>(kb) * 32 + part * (32 / L);
  Raw8<T> r[4 / L];
  load_block<T, VEC>(x + (real ? row : 0) * ldx + k, real ? static_cast<int>(K - k) : 0, r);
  const uint32_t byte = quantize_block<T, FMT, L>(r, c);
  if (part == 0) *scale = static_cast<uint8_t>(byte);  // 0 for a row of the fill
  if (!real) return;
  uint8_t* dst = codes + row * code_pitch + static_cast<int64_t>(kb) * (kWords * L * 4) + part * (kWords * 4);
  if constexpr (kWords == 1) *reinterpret_cast<uint32_t*>(dst) = c[0];
  else if constexpr (kWords == 2) *reinterpret_cast<uint2*>(dst) = make_uint2(c[0], c[1]);
  else {
#pragma unroll
    for (int i = 0; i < kWords; i += 4)
      *reinterpret_cast<uint4*>(dst + 4 * i) = make_uint4(c[i], c[i + 1], c[i + 2], c[i + 3]);
  }
}

// ---------------------------------------------------------------------------------------------------------
// The inverse: half a warp takes the 128 elements of a scale word of kRows neighbouring rows, all loads before the
// arithmetic, and a lane eight elements of each, which it stores at once (25600 x 1536 to fp32 in 30 us, 5.9 TB/s; 43 us
// with two 128-bit stores to a lane, each half a sector).
// ---------------------------------------------------------------------------------------------------------
constexpr int kRows = 4;

template <typename T, int FMT, bool VEC>
__global__ void __launch_bounds__(kThreads) dequantize_kernel(const uint8_t* __restrict__ codes,
                                                              const uint8_t* __restrict__ scales, int64_t rows,
                                                              int64_t K, int64_t items, uint32_t ktiles,
                                                              int64_t code_pitch, T* __restrict__ out) {
  const int64_t item = static_cast<int64_t>(blockIdx.x) * (kThreads / 16) + (threadIdx.x >> 4);
  if (item >= items) return;
  const int64_t group = items <= 0xffffffffll ? static_cast<uint32_t>(item) / ktiles : item / ktiles;
  const int64_t row = group * kRows;
  const uint32_t kt = static_cast<uint32_t>(item - group * ktiles);
  const int lane16 = threadIdx.x & 15;
  const uint8_t* word = scales + scale_word_offset(row, kt, ktiles) + (lane16 >> 2);  // the group's rows: 16 bytes apart
  const int real = static_cast<int>(min(int64_t(kRows), rows - row));
  const int64_t k = static_cast<int64_t>(kt) * 128 + lane16 * 8;
  const int left = static_cast<int>(K - k);
  const uint8_t* code = codes + row * code_pitch + static_cast<int64_t>(kt) * (FMT == KO_MXFP4 ? 64 : 128) +
                        lane16 * (FMT == KO_MXFP4 ? 4 : 8);
  T* dst = out + row * K + k;
  uint2 c[kRows];
  uint32_t byte[kRows];
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    c[i] = make_uint2(0u, 0u);
    byte[i] = 0u;
    if (i < real) {
      byte[i] = __ldg(word + 16 * i);
      if constexpr (FMT == KO_MXFP4) c[i].x = __ldg(reinterpret_cast<const uint32_t*>(code + i * code_pitch));
      else c[i] = __ldg(reinterpret_cast<const uint2*>(code + i * code_pitch));
    }
  }
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    if (i >= real) break;
    const float s = scale_value(byte[i]);
    float v[8];
    if constexpr (FMT == KO_MXFP4) {
      unpack_e2m1x8(c[i].x, v);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 f = unpack_e4m3x2(((j < 2 ? c[i].x : c[i].y) >> (16 * (j & 1))) & 0xffffu);
        v[2 * j] = f.x;
        v[2 * j + 1] = f.y;
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] *= s;
    store8<T, VEC>(dst + i * K, left, v);
  }
}

// ---------------------------------------------------------------------------------------------------------
// A weight [K][N] to its transpose in mxfp4: a thread takes one column of 32 rows, a whole block. Neighbouring threads
// read neighbouring columns; each writes the block's 16 bytes. Once per weight, so the scattered writes stay (8192 x 8192
// bf16 in 116 us, 1.5 TB/s; four blocks to a thread, 64 bytes in a row, took 97, and 384 x 1536 then 11 us instead of 4).
// ---------------------------------------------------------------------------------------------------------
template <typename T>
__global__ void __launch_bounds__(kThreads) pack_weight_kernel(const T* __restrict__ w, int64_t K, int64_t N,
                                                               uint32_t kblocks, int64_t n_blocks,
                                                               int64_t code_pitch, uint8_t* __restrict__ codes,
                                                               uint8_t* __restrict__ scales) {
  const int64_t kb = blockIdx.x % kblocks;
  const int64_t n = static_cast<int64_t>(blockIdx.x / kblocks) * kThreads + threadIdx.x;
  if (n >= n_blocks) return;  // n_blocks: N rounded up to the scale tile's 128
  uint8_t* byte_at = scales + scale_word_offset(n, kb >> 2, kblocks >> 2) + (kb & 3);
  if (n >= N) {
    *byte_at = 0;
    return;
  }
  float v[32];
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    const int64_t k = kb * 32 + i;
    v[i] = k < K ? to_f(w[k * N + n]) : 0.f;
    m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
  }
  const uint32_t byte = scale_byte<KO_MXFP4>(m);
  const float inv = scale_inverse(byte);
  uint32_t c[4];
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    float t[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = v[g * 8 + i];
    c[g] = byte == 255u ? 0u : pack_e2m1x8(t, inv);
  }
  *byte_at = static_cast<uint8_t>(byte);
  *reinterpret_cast<uint4*>(codes + n * code_pitch + kb * 16) = make_uint4(c[0], c[1], c[2], c[3]);
}

// ---------------------------------------------------------------------------------------------------------
// Residual + root-mean-square norm. T threads share a row and keep its NV groups of eight elements each in fp32
// registers from the load to the store, so h and o are read once; the sum of squares is a shuffle tree and, for rows of
// more than a warp, one exchange through shared memory, both in a fixed order. Four lanes hold a block of 32 and sixteen
// the 128 elements of a scale word, so a quantised block costs two shuffles and its scales are stored a word at a time.
// Bound by HBM: 16384 x 8192 bf16 to mxfp8 in 154 us (6.2 TB/s; 68 % of the issue slots), 25664 x 384 fp32 with bias and scale in
// 25.6 us (5.0 TB/s), 23.2 without. Rows that are not whole groups of eight are read and written element by element, neighbouring
// lanes 16 or 32 bytes apart, and bound by that: 16384 x 1001 to mxfp8 in 81 us from fp32 and 57 from bf16 (2.7 and 2.0 TB/s),
// as values in 158 and 86.
// OUT: -1 writes y in the input's type, else the MX format.
// ---------------------------------------------------------------------------------------------------------
// 1 / sqrt(x) as the sum of two fp32 numbers: the special-function value r and one Newton step's correction, r (1 - x r^2)
// / 2, with r^2 kept exactly. y then has the roundings of v * gamma and of the product, and none of r: 5.7e-8 from the exact
// values in the 2-norm (25664 x 384 fp32), as a division in fp32 has it, 6.2e-8 with the rounded 1 / sqrt(x) alone. Most shapes
// take the same time without it, 16384 x 4096 bf16 to mxfp8 76.8 us instead of 79.9. About one 8-bit code in a million, next
// to a border, comes out on its other side either way. Where r^2 could leave the range, r is the rounded value alone.
__device__ __forceinline__ float2 inverse_root(float x) {
  if (!(x > 1e-30f && x < 1e30f)) return make_float2(1.0f / sqrtf(x), 0.f);
  const float r = rsqrtf(x), t = r * r;
  const float rest = fmaf(-x, t, 1.0f) - x * fmaf(r, r, -t);
  return make_float2(r, 0.5f * r * rest);
}
__device__ __forceinline__ float scaled(float p, float2 r) { return fmaf(p, r.y, p * r.x); }

struct NormArgs {
  const void *h, *o, *bias, *scale, *gamma;
  void *h_out, *y;
  uint8_t *codes, *scales;
  int64_t ldh, ldo, rows, C, code_pitch, grid_rows;
  uint32_t ktiles;
  float eps;
};

template <typename T, int OUT, bool VEC, int TPR, int NV>
__global__ void __launch_bounds__(TPR > kThreads ? TPR : kThreads) rmsnorm_kernel(const NormArgs a) {
  constexpr int kBlock = TPR > kThreads ? TPR : kThreads;
  constexpr int kBlockRows = kBlock / TPR;
  constexpr int kWarps = TPR / 32;  // warps of a row (0: half a warp)
  __shared__ float part[kBlock / 32];
  const int t = threadIdx.x % TPR;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kBlockRows + threadIdx.x / TPR;
  const bool real = row < a.rows;
  const int left = real ? static_cast<int>(a.C) - t * 8 : 0;  // elements from this thread's first one to the row's end
  constexpr int kStep = TPR * 8;
  // All loads of a row go out before the arithmetic, gamma's while the sum is taken. The widest rows of fp32 have no
  // registers for that with the block's 1024 threads: they take group after group (2048 x 32768: 171 us, 470 otherwise).
  constexpr bool kAhead = !(sizeof(T) == 4 && TPR * NV > 2048);
  constexpr int kHold = kAhead ? NV : 1;
  float v[NV][8];
  Raw8<T> g[kHold];
  auto group = [&](const void* p, int i) {
    return load8<T, VEC>(static_cast<const T*>(p) + t * 8 + i * kStep, left - i * kStep);
  };
  {
    const T* h = static_cast<const T*>(a.h) + row * a.ldh;
    const T* o = a.o ? static_cast<const T*>(a.o) + row * a.ldo : nullptr;
    // v[i], the widened o, becomes (o + bias) * scale for the groups [from, to); one branch for all of them
    auto affine = [&](auto from, auto to) {
      float x[8];
      if (a.bias) {
#pragma unroll
        for (int i = from; i < to; ++i) {
          widen8(group(a.bias, i), x);
#pragma unroll
          for (int j = 0; j < 8; ++j) v[i][j] += x[j];
        }
      }
      if (a.scale) {
#pragma unroll
        for (int i = from; i < to; ++i) {
          widen8(group(a.scale, i), x);
#pragma unroll
          for (int j = 0; j < 8; ++j) v[i][j] *= x[j];
        }
      }
    };
    auto add = [&](int i, const Raw8<T>& hr) {
      float x[8];
      widen8(hr, x);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] += x[j];
    };
    if constexpr (kAhead) {
      Raw8<T> r[NV], q[NV];
#pragma unroll
      for (int i = 0; i < NV; ++i) r[i] = group(h, i);
      if (o) {
#pragma unroll
        for (int i = 0; i < NV; ++i) q[i] = group(o, i);
#pragma unroll
        for (int i = 0; i < NV; ++i) widen8(q[i], v[i]);
        affine(0, NV);
#pragma unroll
        for (int i = 0; i < NV; ++i) add(i, r[i]);
      } else {
#pragma unroll
        for (int i = 0; i < NV; ++i) widen8(r[i], v[i]);
      }
#pragma unroll
      for (int i = 0; i < NV; ++i) g[i] = group(a.gamma, i);
    } else {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const Raw8<T> r = group(h, i);
        if (o) {
          widen8(group(o, i), v[i]);
          affine(i, i + 1);
          add(i, r);
        } else {
          widen8(r, v[i]);
        }
      }
    }
  }
  auto gamma_of = [&](int i) {
    if constexpr (kAhead) return g[i];
    else return group(a.gamma, i);
  };
  if (a.h_out) {
    T* h_out = static_cast<T*>(a.h_out) + row * a.C + t * 8;
#pragma unroll
    for (int i = 0; i < NV; ++i) store8<T, VEC>(h_out + i * kStep, left - i * kStep, v[i]);
  }
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i)
    sum += ((v[i][0] * v[i][0] + v[i][1] * v[i][1]) + (v[i][2] * v[i][2] + v[i][3] * v[i][3])) +
           ((v[i][4] * v[i][4] + v[i][5] * v[i][5]) + (v[i][6] * v[i][6] + v[i][7] * v[i][7]));
#pragma unroll
  for (int s = (TPR < 32 ? TPR : 32) / 2; s > 0; s >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
  if constexpr (kWarps > 1) {
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = sum;
    __syncthreads();
    const int w0 = (threadIdx.x / TPR) * kWarps;
    sum = (threadIdx.x & 31) < kWarps ? part[w0 + (threadIdx.x & 31)] : 0.f;
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
  }
  const float2 rstd = inverse_root(sum / static_cast<float>(a.C) + a.eps);
  if constexpr (OUT < 0) {
    if (!real) return;
    T* y = static_cast<T*>(a.y) + row * a.C + t * 8;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float gm[8];
      widen8(gamma_of(i), gm);
#pragma unroll
      for (int j = 0; j < 8; ++j) gm[j] = scaled(v[i][j] * gm[j], rstd);
      store8<T, VEC>(y + i * kStep, left - i * kStep, gm);
    }
  } else {
    if (row >= a.grid_rows) return;
    uint8_t* word = a.scales + scale_word_offset(row, t >> 4, a.ktiles);  // a k tile is 512 bytes
    constexpr int kBytes = OUT == KO_MXFP4 ? 4 : 8;
    uint8_t* code = a.codes + row * a.code_pitch + t * kBytes;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if ((t >> 4) + i * (TPR / 16) >= static_cast<int>(a.ktiles)) break;  // the same for the sixteen lanes of a group
      if (!real) {
        if ((t & 15) == 0) *reinterpret_cast<uint32_t*>(word + i * (TPR / 16) * 512) = 0u;
        continue;
      }
      float gm[8];
      widen8(gamma_of(i), gm);
      // beyond C v is 0, and 0 * rstd would be NaN for an infinite rstd (eps 0, a row of zeros)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        gm[j] = scaled(v[i][j] * gm[j], rstd);
        if (VEC ? left - i * kStep <= 0 : j >= left - i * kStep) gm[j] = 0.f;
      }
      quantize_group<OUT>(gm, amax_bits8(gm), 0xffffu << (threadIdx.x & 16), code + i * TPR * kBytes,
                          word + i * (TPR / 16) * 512);
    }
  }
}

template <typename T, int OUT, bool VEC, int TPR, int NV>
int launch_norm(const NormArgs& a, cudaStream_t s) {
  constexpr int kBlock = TPR > kThreads ? TPR : kThreads;
  const int64_t blocks = (a.grid_rows + kBlock / TPR - 1) / (kBlock / TPR);
  if (blocks > 0x7fffffff) return ko::fail(KO_ERR_INVALID_ARGUMENT, "ko_residual_rmsnorm: too many rows");
  rmsnorm_kernel<T, OUT, VEC, TPR, NV><<<static_cast<unsigned>(blocks), kBlock, 0, s>>>(a);
  return ko::check_launch("ko_residual_rmsnorm");
}

template <typename T, int OUT, bool VEC>
int pick_norm(const NormArgs& a, cudaStream_t s) {
  // Half a warp to a row up to 384 (102656 x 384 in 76 us fp32 and 44 us bf16; 75 and 54 with a warp of two groups to a
  // thread), with no more groups than the row has. Then two groups of eight to a thread: 16384 x 4096 in 127 us fp32 and
  // 78 us bf16, 130 and 80 with half the threads, 127 and 92 with twice as many; one row of 4096 in 2.4 us, 2.8 and 2.4.
  // From 8192 on the threads of a block bound it: 8192 x 16384 bf16 in 148 us with 512 threads and four groups, 212 with
  // 1024 and two. 1024 threads leave 64 registers each, and rows over 16384 that are read element by element do not fit: 16-bit
  // ones spill 60 to 92 bytes, fp32 ones 4.
  if (a.C <= 128) return launch_norm<T, OUT, VEC, 16, 1>(a, s);
  if (a.C <= 256) return launch_norm<T, OUT, VEC, 16, 2>(a, s);
  if (a.C <= 384) return launch_norm<T, OUT, VEC, 16, 3>(a, s);
  if (a.C <= 512) return launch_norm<T, OUT, VEC, 32, 2>(a, s);
  if (a.C <= 1024) return launch_norm<T, OUT, VEC, 64, 2>(a, s);
  if (a.C <= 2048) return launch_norm<T, OUT, VEC, 128, 2>(a, s);
  if (a.C <= 4096) return launch_norm<T, OUT, VEC, 256, 2>(a, s);
  if (a.C <= 8192) return launch_norm<T, OUT, VEC, 512, 2>(a, s);
  if (a.C <= 16384) return launch_norm<T, OUT, VEC, 512, 4>(a, s);
  return launch_norm<T, OUT, VEC, 1024, 4>(a, s);
}

template <typename T>
int dispatch_norm(const NormArgs& a, int out, bool vec, cudaStream_t s) {
  if (out < 0) return vec ? pick_norm<T, -1, true>(a, s) : pick_norm<T, -1, false>(a, s);
  if (out == KO_MXFP4) return vec ? pick_norm<T, KO_MXFP4, true>(a, s) : pick_norm<T, KO_MXFP4, false>(a, s);
  return vec ? pick_norm<T, KO_MXFP8, true>(a, s) : pick_norm<T, KO_MXFP8, false>(a, s);
}

template <typename T, int FMT>
int launch_quantize(const void* x, int64_t rows, int64_t K, int64_t ldx, void* codes, void* scales, bool vec,
                    cudaStream_t s) {
  const int64_t kblocks = padded_k(K) / 32, items = (rows + 127) / 128 * 128 * kblocks;
  auto go = [&](auto kernel, int lanes) {
    const int64_t blocks = (items * lanes + kThreads - 1) / kThreads;
    if (blocks > 0x7fffffff) return ko::fail(KO_ERR_INVALID_ARGUMENT, "ko_quantize_mx: too many elements");
    kernel<<<static_cast<unsigned>(blocks), kThreads, 0, s>>>(
        static_cast<const T*>(x), rows, K, ldx, items, static_cast<uint32_t>(kblocks), code_pitch(K, FMT),
        static_cast<uint8_t*>(codes), static_cast<uint8_t*>(scales));
    return ko::check_launch("ko_quantize_mx");
  };
  if (!vec) return go(quantize_kernel<T, FMT, false, 4>, 4);
  constexpr int L = sizeof(T) == 2 ? 1 : 2;
  return go(quantize_kernel<T, FMT, true, L>, L);
}

template <typename T>
int launch_dequantize(const void* codes, const void* scales, int fmt, int64_t rows, int64_t K, void* out,
                      cudaStream_t s) {
  const int64_t ktiles = padded_k(K) / 128, items = (rows + kRows - 1) / kRows * ktiles;
  const int64_t blocks = (items + kThreads / 16 - 1) / (kThreads / 16);
  if (blocks > 0x7fffffff) return ko::fail(KO_ERR_INVALID_ARGUMENT, "ko_dequantize_mx: too many elements");
  const bool vec = reinterpret_cast<uintptr_t>(out) % (8 * sizeof(T)) == 0 && K % 8 == 0;
  const uint8_t *c = static_cast<const uint8_t*>(codes), *sc = static_cast<const uint8_t*>(scales);
  auto go = [&](auto kernel) {
    kernel<<<static_cast<unsigned>(blocks), kThreads, 0, s>>>(c, sc, rows, K, items, static_cast<uint32_t>(ktiles),
                                                              code_pitch(K, fmt), static_cast<T*>(out));
  };
  if (fmt == KO_MXFP4) go(vec ? dequantize_kernel<T, KO_MXFP4, true> : dequantize_kernel<T, KO_MXFP4, false>);
  else go(vec ? dequantize_kernel<T, KO_MXFP8, true> : dequantize_kernel<T, KO_MXFP8, false>);
  return ko::check_launch("ko_dequantize_mx");
}

bool aligned_to(const void* p, int64_t n) { return reinterpret_cast<uintptr_t>(p) % static_cast<uintptr_t>(n) == 0; }

}  // namespace

extern "C" int64_t ko_mx_codes_bytes(int64_t rows, int64_t K, int fmt) {
  if (rows < 0 || rows > kMaxRows || K < 1 || K > kMaxK || !fmt_ok(fmt)) return -1;
  return rows * code_pitch(K, fmt);
}
extern "C" int64_t ko_mx_scales_bytes(int64_t rows, int64_t K) {
  if (rows < 0 || rows > kMaxRows || K < 1 || K > kMaxK) return -1;
  return (rows + 127) / 128 * 128 * (padded_k(K) / 32);
}

extern "C" int ko_quantize_mx(const void* x, int dtype, int64_t rows, int64_t K, int64_t ldx, int fmt, void* codes,
                              void* scales, ko_stream_t stream) {
  const std::string who = "ko_quantize_mx: ";
  if (rows < 0 || rows > kMaxRows || K < 1 || K > kMaxK || ldx < K)
    return ko::fail(KO_ERR_INVALID_ARGUMENT, who + "need 0 <= rows <= 2^31, 1 <= K <= 2^24 and ldx >= K");
  if (!extent_ok(rows, ldx)) return ko::fail(KO_ERR_INVALID_ARGUMENT, who + "the rows' pitch spans more than 2^46 elements");
  if (!dtype_ok(dtype) || !fmt_ok(fmt)) return ko::fail(KO_ERR_INVALID_ARGUMENT, who + "unknown element type or format");
  if (rows == 0) return KO_OK;
  if (!x || !codes || !scales) return ko::fail(KO_ERR_INVALID_ARGUMENT, who + "null pointer");
  const int64_t es = dtype_size(dtype);
  if (!aligned_to(x, es) || !ko::aligned16(codes) || !ko::aligned16(scales))
    return ko::fail(KO_ERR_INVALID_ARGUMENT, who + "x must be aligned to its elements, codes and scales to 16 bytes");
  const Range in = span_of(x, rows, ldx, K, es), c = {codes, ko_mx_codes_bytes(rows, K, fmt)},
              sc = {scales, ko_mx_scales_bytes(rows, K)};
  if (meets(c, {in, sc}) || meets(sc, {in}))
    return ko::fail(KO_ERR_INVALID_ARGUMENT, who + "codes or scales overlap x or each other");
  const bool vec = groups_of_8(x, dtype, ldx, K);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const bool f4 = fmt == KO_MXFP4;
  if (dtype == KO_F32)
    return f4 ? launch_quantize<float, KO_MXFP4>(x, rows, K, ldx, codes, scales, vec, s)
              : launch_quantize<float, KO_MXFP8>(x, rows, K, ldx, codes, scales, vec, s);
  if (dtype == KO_BF16)
    return f4 ? launch_quantize<__nv_bfloat16, KO_MXFP4>(x, rows, K, ldx, codes, scales, vec, s)
              : launch_quantize<__nv_bfloat16, KO_MXFP8>(x, rows, K, ldx, codes, scales, vec, s);
  return f4 ? launch_quantize<__half, KO_MXFP4>(x, rows, K, ldx, codes, scales, vec, s)
            : launch_quantize<__half, KO_MXFP8>(x, rows, K, ldx, codes, scales, vec, s);
}

extern "C" int ko_dequantize_mx(const void* codes, const void* scales, int fmt, int64_t rows, int64_t K, void* out,
                                int dtype, ko_stream_t stream) {
  const std::string who = "ko_dequantize_mx: ";
  if (rows < 0 || rows > kMaxRows || K < 1 || K > kMaxK)
    return ko::fail(KO_ERR_INVALID_ARGUMENT, who + "need 0 <= rows <= 2^31 and 1 <= K <= 2^24");
  if (!dtype_ok(dtype) || !fmt_ok(fmt)) return ko::fail(KO_ERR_INVALID_ARGUMENT, who + "unknown element type or format");
  if (rows == 0) return KO_OK;
  if (!codes || !scales || !out) return ko::fail(KO_ERR_INVALID_ARGUMENT, who + "null pointer");
  if (!ko::aligned16(codes) || !ko::aligned16(scales) || !aligned_to(out, dtype_size(dtype)))
    return ko::fail(KO_ERR_INVALID_ARGUMENT, who + "codes and scales must be 16-byte aligned, out to its elements");
  if (meets({out, rows * K * dtype_size(dtype)},
            {{codes, ko_mx_codes_bytes(rows, K, fmt)}, {scales, ko_mx_scales_bytes(rows, K)}}))
    return ko::fail(KO_ERR_INVALID_ARGUMENT, who + "out overlaps codes or scales");
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == KO_F32) return launch_dequantize<float>(codes, scales, fmt, rows, K, out, s);
  if (dtype == KO_BF16) return launch_dequantize<__nv_bfloat16>(codes, scales, fmt, rows, K, out, s);
  return launch_dequantize<__half>(codes, scales, fmt, rows, K, out, s);
}

extern "C" int ko_pack_weight_mxfp4(const void* w, int dtype, int64_t K, int64_t N, void* codes, void* scales,
                                    ko_stream_t stream) {
  const std::string who = "ko_pack_weight_mxfp4: ";
  if (K < 1 || K > kMaxK || N < 1 || N > kMaxRows)
    return ko::fail(KO_ERR_INVALID_ARGUMENT, who + "need 1 <= K <= 2^24 and 1 <= N <= 2^31");
  if (!dtype_ok(dtype)) return ko::fail(KO_ERR_INVALID_ARGUMENT, who + "unknown element type");
  if (!w || !codes || !scales) return ko::fail(KO_ERR_INVALID_ARGUMENT, who + "null pointer");
  if (!aligned_to(w, dtype_size(dtype)) || !ko::aligned16(codes) || !ko::aligned16(scales))
    return ko::fail(KO_ERR_INVALID_ARGUMENT, who + "w must be aligned to its elements, codes and scales to 16 bytes");
  const Range in = {w, K * N * dtype_size(dtype)}, out = {codes, ko_mx_codes_bytes(N, K, KO_MXFP4)},
              tiles = {scales, ko_mx_scales_bytes(N, K)};
  if (meets(out, {in, tiles}) || meets(tiles, {in}))
    return ko::fail(KO_ERR_INVALID_ARGUMENT, who + "codes or scales overlap w or each other");
  const int64_t kblocks = padded_k(K) / 32, n_rows = (N + 127) / 128 * 128;
  const int64_t blocks = kblocks * ((n_rows + kThreads - 1) / kThreads);
  if (blocks > 0x7fffffff) return ko::fail(KO_ERR_INVALID_ARGUMENT, who + "the weight is too large");
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const unsigned g = static_cast<unsigned>(blocks);
  uint8_t *c = static_cast<uint8_t*>(codes), *sc = static_cast<uint8_t*>(scales);
  const int64_t pitch = code_pitch(K, KO_MXFP4);
  const uint32_t kb = static_cast<uint32_t>(kblocks);
  if (dtype == KO_F32)
    pack_weight_kernel<float><<<g, kThreads, 0, s>>>(static_cast<const float*>(w), K, N, kb, n_rows, pitch, c, sc);
  else if (dtype == KO_BF16)
    pack_weight_kernel<__nv_bfloat16><<<g, kThreads, 0, s>>>(static_cast<const __nv_bfloat16*>(w), K, N, kb, n_rows,
                                                             pitch, c, sc);
  else
    pack_weight_kernel<__half><<<g, kThreads, 0, s>>>(static_cast<const __half*>(w), K, N, kb, n_rows, pitch, c, sc);
  return ko::check_launch("ko_pack_weight_mxfp4");
}

extern "C" int ko_residual_rmsnorm(const void* h, int64_t ldh, const void* o, int64_t ldo, const void* bias,
                                   const void* scale, const void* gamma, int dtype, float eps, int64_t rows,
                                   int64_t C, void* h_out, void* y, int fmt, void* codes, void* scales,
                                   ko_stream_t stream) {
  const std::string who = "ko_residual_rmsnorm: ";
  if (rows < 0 || rows > kMaxRows || C < 1 || C > 32768 || ldh < C || (o && ldo < C))
    return ko::fail(KO_ERR_INVALID_ARGUMENT, who + "need 0 <= rows <= 2^31, 1 <= C <= 32768 and pitches of at least C");
  if (!extent_ok(rows, ldh) || (o && !extent_ok(rows, ldo)))
    return ko::fail(KO_ERR_INVALID_ARGUMENT, who + "the rows' pitch spans more than 2^46 elements");
  if (!dtype_ok(dtype)) return ko::fail(KO_ERR_INVALID_ARGUMENT, who + "unknown element type");
  if (!(eps >= 0.f)) return ko::fail(KO_ERR_INVALID_ARGUMENT, who + "eps must not be negative");
  if (y ? (codes || scales) : (!codes || !scales || !fmt_ok(fmt)))
    if (rows > 0 || (y && (codes || scales)))
      return ko::fail(KO_ERR_INVALID_ARGUMENT, who + "give either y, or codes and scales with a known format");
  if (rows == 0) return KO_OK;
  if (!h || !gamma) return ko::fail(KO_ERR_INVALID_ARGUMENT, who + "null pointer");
  if (!o && (bias || scale))
    return ko::fail(KO_ERR_INVALID_ARGUMENT, who + "bias and scale belong to o");
  // A row of h and o is read whole before it is written, by the threads that write it: h_out or y in place of one of them is
  // fine. Every other overlap of an output is not: with another row, with the vectors, that all rows read, or with another
  // output.
  const int64_t es = dtype_size(dtype), out_bytes = rows * C * es;
  const Range hs = span_of(h, rows, ldh, C, es), os = span_of(o, rows, o ? ldo : C, C, es);
  const Range vs[] = {{bias, C * es}, {scale, C * es}, {gamma, C * es}};
  const Range ho = {h_out, out_bytes}, yo = {y, out_bytes}, co = {codes, y ? 0 : ko_mx_codes_bytes(rows, C, fmt)},
              so = {scales, y ? 0 : ko_mx_scales_bytes(rows, C)};
  auto meets_rows = [&](const Range& out, const Range& in, int64_t pitch) {
    return !(in.p == out.p && (rows == 1 || pitch == C)) && meets(out, {in});
  };
  if (meets_rows(ho, hs, ldh) || meets_rows(ho, os, ldo) || meets_rows(yo, hs, ldh) || meets_rows(yo, os, ldo) ||
      meets(co, {hs, os, so, vs[0], vs[1], vs[2]}) || meets(so, {hs, os, vs[0], vs[1], vs[2]}) ||
      meets(ho, {yo, co, so, vs[0], vs[1], vs[2]}) || meets(yo, {vs[0], vs[1], vs[2]}))
    return ko::fail(KO_ERR_INVALID_ARGUMENT, who + "an output overlaps an input or another output (h_out or y may be h or o "
                                                   "itself, the same contiguous rows)");
  bool vec = ldh % 8 == 0 && (!o || ldo % 8 == 0);
  const void* elems[] = {h, o, bias, scale, gamma, h_out, y};
  for (const void* p : elems) {
    if (p && !aligned_to(p, es)) return ko::fail(KO_ERR_INVALID_ARGUMENT, who + "a pointer is not aligned to its elements");
    vec = vec && groups_of_8(p, dtype, C, C);
  }
  if (!y && (!ko::aligned16(codes) || !ko::aligned16(scales)))
    return ko::fail(KO_ERR_INVALID_ARGUMENT, who + "codes and scales must be 16-byte aligned");
  NormArgs a{};
  a.h = h;
  a.o = o;
  a.bias = bias;
  a.scale = scale;
  a.gamma = gamma;
  a.h_out = h_out;
  a.y = y;
  a.codes = static_cast<uint8_t*>(codes);
  a.scales = static_cast<uint8_t*>(scales);
  a.ldh = ldh;
  a.ldo = ldo;
  a.rows = rows;
  a.C = C;
  a.code_pitch = y ? 0 : code_pitch(C, fmt);
  a.grid_rows = y ? rows : (rows + 127) / 128 * 128;
  a.ktiles = static_cast<uint32_t>(padded_k(C) / 128);
  a.eps = eps;
  const int out = y ? -1 : fmt;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == KO_F32) return dispatch_norm<float>(a, out, vec, s);
  if (dtype == KO_BF16) return dispatch_norm<__nv_bfloat16>(a, out, vec, s);
  return dispatch_norm<__half>(a, out, vec, s);
}
