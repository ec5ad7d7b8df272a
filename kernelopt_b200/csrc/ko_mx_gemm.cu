// Product of microscaled operands:  out[M][N] = act(A[M][K] @ W[N][K]^T + bias),  A in mxfp4 or mxfp8, W in mxfp4.
// Formats and layout: ko_mx.cuh.
//
// 64 x 64 tiles: 256 threads expand 32 elements along K of both operands to fp32 in shared memory and accumulate
// 4 x 4 outputs each in fp32.
#include <string>

#include "ko_mx.cuh"

namespace {

using namespace komx;

constexpr int kTile = 64;
constexpr int kThreads = 256;

__device__ __forceinline__ float act_f(float v, int act) {
  // 1 + erf(v / sqrt 2) as erfc(-v / sqrt 2), which keeps its relative accuracy where v is far below zero
  if (act == KO_ACT_GELU) return 0.5f * v * erfcf(v * -0.7071067811865476f);
  if (act == KO_ACT_RELU) return v < 0.f ? 0.f : v;
  return v;
}

template <int FMT>
__device__ __forceinline__ void expand8(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                                        int64_t row, int64_t rows, int64_t pitch, int64_t ktiles, int64_t k,
                                        float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = 0.f;
  if (row >= rows) return;
  const float s = scale_value(scales[scale_word_offset(row, k >> 7, ktiles) + ((k >> 5) & 3)]);
  if constexpr (FMT == KO_MXFP4) {
    unpack_e2m1x8(*reinterpret_cast<const uint32_t*>(codes + row * pitch + k / 2), v);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = unpack_e4m3x2(*reinterpret_cast<const uint16_t*>(codes + row * pitch + k + 2 * i));
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] *= s;
}

template <int FMT, typename T>
__global__ void __launch_bounds__(kThreads)
    linear_kernel(const uint8_t* __restrict__ ac, const uint8_t* __restrict__ as, const uint8_t* __restrict__ wc,
                  const uint8_t* __restrict__ ws, const float* __restrict__ bias, int64_t M, int64_t N, int64_t Kp,
                  int act, T* __restrict__ out, int64_t n_tiles) {
  __shared__ float sa[32][kTile + 1], sw[32][kTile + 1];
  const int64_t m0 = blockIdx.x / n_tiles * kTile, n0 = blockIdx.x % n_tiles * kTile;
  const int lr = threadIdx.x >> 2, lk = (threadIdx.x & 3) * 8;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int64_t a_pitch = FMT == KO_MXFP4 ? Kp / 2 : Kp;
  float acc[4][4] = {};
  for (int64_t k0 = 0; k0 < Kp; k0 += 32) {
    float v[8];
    expand8<FMT>(ac, as, m0 + lr, M, a_pitch, Kp / 128, k0 + lk, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) sa[lk + i][lr] = v[i];
    expand8<KO_MXFP4>(wc, ws, n0 + lr, N, Kp / 2, Kp / 128, k0 + lk, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) sw[lk + i][lr] = v[i];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 32; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(sa[k][ty + 16 * i], sw[k][tx + 16 * j], acc[i][j]);
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t m = m0 + ty + 16 * i, n = n0 + tx + 16 * j;
      if (m < M && n < N) out[m * N + n] = from_f<T>(act_f(acc[i][j] + (bias ? bias[n] : 0.f), act));
    }
}

template <int FMT>
int launch(const uint8_t* ac, const uint8_t* as, const uint8_t* wc, const uint8_t* ws, const float* bias, int64_t M,
           int64_t K, int64_t N, int act, void* out, int dtype, cudaStream_t s) {
  const int64_t n_tiles = (N + kTile - 1) / kTile, blocks = (M + kTile - 1) / kTile * n_tiles, Kp = padded_k(K);
  if (blocks > 0x7fffffff) return ko::fail(KO_ERR_INVALID_ARGUMENT, "ko_linear_mxfp4: the output is too large");
  const unsigned g = static_cast<unsigned>(blocks);
  if (dtype == KO_F32)
    linear_kernel<FMT><<<g, kThreads, 0, s>>>(ac, as, wc, ws, bias, M, N, Kp, act, static_cast<float*>(out), n_tiles);
  else if (dtype == KO_BF16)
    linear_kernel<FMT><<<g, kThreads, 0, s>>>(ac, as, wc, ws, bias, M, N, Kp, act, static_cast<__nv_bfloat16*>(out),
                                              n_tiles);
  else
    linear_kernel<FMT><<<g, kThreads, 0, s>>>(ac, as, wc, ws, bias, M, N, Kp, act, static_cast<__half*>(out), n_tiles);
  return ko::check_launch("ko_linear_mxfp4");
}

}  // namespace

extern "C" int ko_linear_mxfp4(const void* a_codes, const void* a_scales, int a_fmt, const void* w_codes,
                               const void* w_scales, const float* bias, int64_t M, int64_t K, int64_t N, int act,
                               void* out, int out_dtype, int* dev_status, ko_stream_t stream) {
  const std::string who = "ko_linear_mxfp4: ";
  if (M < 0 || M > kMaxRows || K < 1 || K > kMaxK || N < 1 || N > kMaxRows)
    return ko::fail(KO_ERR_INVALID_ARGUMENT, who + "need 0 <= M <= 2^31, 1 <= K <= 2^24 and 1 <= N <= 2^31");
  if (!fmt_ok(a_fmt) || !dtype_ok(out_dtype))
    return ko::fail(KO_ERR_INVALID_ARGUMENT, who + "unknown format or output type");
  if (act != KO_ACT_NONE && act != KO_ACT_GELU && act != KO_ACT_RELU)
    return ko::fail(KO_ERR_INVALID_ARGUMENT, who + "act must be KO_ACT_NONE, KO_ACT_GELU or KO_ACT_RELU");
  if (M == 0) return KO_OK;
  if (!a_codes || !a_scales || !w_codes || !w_scales || !out)
    return ko::fail(KO_ERR_INVALID_ARGUMENT, who + "null pointer");
  if (!ko::aligned16(a_codes) || !ko::aligned16(a_scales) || !ko::aligned16(w_codes) || !ko::aligned16(w_scales))
    return ko::fail(KO_ERR_INVALID_ARGUMENT, who + "codes and scales must be 16-byte aligned");
  if (reinterpret_cast<uintptr_t>(out) % static_cast<uintptr_t>(dtype_size(out_dtype)) != 0 ||
      reinterpret_cast<uintptr_t>(bias) % 4 != 0)
    return ko::fail(KO_ERR_INVALID_ARGUMENT, who + "out and bias must be aligned to their elements");
  const uint8_t *ac = static_cast<const uint8_t*>(a_codes), *as = static_cast<const uint8_t*>(a_scales);
  const uint8_t *wc = static_cast<const uint8_t*>(w_codes), *ws = static_cast<const uint8_t*>(w_scales);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  (void)dev_status;
  return a_fmt == KO_MXFP4 ? launch<KO_MXFP4>(ac, as, wc, ws, bias, M, K, N, act, out, out_dtype, s)
                           : launch<KO_MXFP8>(ac, as, wc, ws, bias, M, K, N, act, out, out_dtype, s);
}
