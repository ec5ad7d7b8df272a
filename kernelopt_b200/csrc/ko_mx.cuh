// Microscaled (OCP MX) data as the library lays it out, and the conversions its kernels share.
//
// A matrix [rows][K] in an MX format is, with Kp = K rounded up to a multiple of 128:
//   codes   mxfp4: [rows][Kp / 2] bytes, element 2i in the low nibble of byte i;  mxfp8: [rows][Kp] bytes
//   scales  [ceil(rows / 128)][Kp / 128][32][4][4] bytes: the e8m0 scale of row 128 R + 32 j + i and block 4 T + b is
//           byte (i, j, b) of tile (R, T). One tile is the 512 contiguous bytes that the block-scaled tensor-core
//           products take as one operand: 32 tensor-memory lanes of 16 bytes, one 32-bit column per group of 32 rows.
// Codes and scales beyond K are zero (scale byte 0, 2^-127), and so are the scales of the rows that fill the last tile.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <initializer_list>

#include "ko_common.cuh"

namespace komx {

inline int64_t padded_k(int64_t K) { return (K + 127) / 128 * 128; }
inline int64_t code_pitch(int64_t K, int fmt) { return fmt == KO_MXFP4 ? padded_k(K) / 2 : padded_k(K); }
inline bool fmt_ok(int fmt) { return fmt == KO_MXFP4 || fmt == KO_MXFP8; }
inline bool dtype_ok(int dt) { return dt == KO_F32 || dt == KO_BF16 || dt == KO_F16; }
inline int64_t dtype_size(int dt) { return dt == KO_F32 ? 4 : 2; }
// Whether rows of `dtype` at p, `pitch` elements apart and `width` long, are whole groups of eight that one access moves.
inline bool groups_of_8(const void* p, int dtype, int64_t pitch, int64_t width) {
  const int64_t group = 8 * dtype_size(dtype);
  return reinterpret_cast<uintptr_t>(p) % static_cast<uintptr_t>(group) == 0 && pitch % 8 == 0 && width % 8 == 0;
}
// Bounds of the entry points: rows times K is at most 2^55, and what rows and their pitch span (extent_ok) 2^46 elements, more
// than an address space holds, so that every size, offset and end address in bytes stays inside 62 bits.
constexpr int64_t kMaxRows = int64_t(1) << 31;
constexpr int64_t kMaxK = int64_t(1) << 24;
constexpr int64_t kMaxExtent = int64_t(1) << 46;
inline bool extent_ok(int64_t rows, int64_t pitch) { return rows <= 1 || pitch <= kMaxExtent / rows; }
// What an output may not share a byte with: the threads that write it are not those that read the others.
struct Range {
  const void* p;
  int64_t bytes;
};
inline Range span_of(const void* p, int64_t rows, int64_t pitch, int64_t width, int64_t size) {
  return {p, ((rows - 1) * pitch + width) * size};
}
inline bool meets(const Range& out, std::initializer_list<Range> others) {
  for (const Range& r : others)
    if (ko::ranges_meet(out.p, out.bytes, r.p, r.bytes)) return true;
  return false;
}

#if defined(__CUDACC__)

// Programmatic dependent launch: a kernel that is launched behind another one may set itself up while the other's last CTAs
// run, and waits here, before it touches global memory, until that grid is complete and what it wrote is visible.
__device__ __forceinline__ void wait_for_previous_grid() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
// Lets such a kernel be launched once every CTA of this grid has come here.
__device__ __forceinline__ void let_next_grid_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

template <typename T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_f<__half>(__half v) { return __half2float(v); }
// One rounding (to nearest even) from fp32 to the output's type.
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }

// Eight consecutive elements as they lie in memory, moved by one access of 256 bits (fp32) or 128 (bf16, fp16). Two
// 128-bit accesses of a lane's 32 bytes would each touch half of every 32-byte sector: the fp32 stores of 25600 x 1536
// dequantised values took 43 us that way.
template <typename T>
struct alignas(16) Raw8 {
  uint32_t w[2 * sizeof(T)];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < static_cast<int>(2 * sizeof(T)); ++i) w[i] = 0u;
  }
};
__device__ __forceinline__ void widen8(const Raw8<float>& r, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(r.w[i]);
}
__device__ __forceinline__ void widen8(const Raw8<__nv_bfloat16>& r, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {  // a bf16 is the upper half of its fp32
    v[2 * i] = __uint_as_float(r.w[i] << 16);
    v[2 * i + 1] = __uint_as_float(r.w[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ void widen8(const Raw8<__half>& r, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&r.w[i]));
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}
template <typename T> __device__ __forceinline__ uint32_t pack2(float a, float b);
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 p = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&p);
}
template <> __device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  const __half2 p = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&p);
}
template <typename T>
__device__ __forceinline__ Raw8<T> narrow8(const float (&v)[8]) {
  Raw8<T> r;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 8; ++i) r.w[i] = __float_as_uint(v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) r.w[i] = pack2<T>(v[2 * i], v[2 * i + 1]);
  }
  return r;
}

// The group of eight elements at `p`, of which `left` (any integer) lie before the end of the row; the others are zero.
// VEC: the row starts on a multiple of a group's bytes and its length is a multiple of 8, so a group is whole or beyond
// the end.
template <typename T, bool VEC>
__device__ __forceinline__ Raw8<T> load8(const T* p, int left) {
  Raw8<T> r;
  r.clear();
  if (VEC) {
    if (left > 0) {
      if constexpr (sizeof(T) == 4) {
        asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=r"(r.w[0]), "=r"(r.w[1]), "=r"(r.w[2]), "=r"(r.w[3]), "=r"(r.w[4]), "=r"(r.w[5]), "=r"(r.w[6]),
                       "=r"(r.w[7])
                     : "l"(p));
      } else {
        const uint4 a = *reinterpret_cast<const uint4*>(p);
        r.w[0] = a.x; r.w[1] = a.y; r.w[2] = a.z; r.w[3] = a.w;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < left) reinterpret_cast<T*>(r.w)[i] = p[i];
  }
  return r;
}
template <typename T, bool VEC>
__device__ __forceinline__ void store8(T* p, int left, const float (&v)[8]) {
  if (VEC) {
    if (left > 0) {
      const Raw8<T> r = narrow8<T>(v);
      if constexpr (sizeof(T) == 4)
        asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(r.w[0]), "r"(r.w[1]),
                     "r"(r.w[2]), "r"(r.w[3]), "r"(r.w[4]), "r"(r.w[5]), "r"(r.w[6]), "r"(r.w[7])
                     : "memory");
      else
        *reinterpret_cast<uint4*>(p) = make_uint4(r.w[0], r.w[1], r.w[2], r.w[3]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < left) p[i] = from_f<T>(v[i]);
  }
}

// Largest magnitude of eight values as the bits of an fp32: ordered like the magnitudes, with infinity and then NaN
// above every finite value, so that one integer maximum also finds what is not finite. The 16-bit types are compared two
// at a time in their own bits, which are ordered the same way.
__device__ __forceinline__ uint32_t amax_bits8(const float (&v)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
  return m;
}
__device__ __forceinline__ uint32_t amax_bits8(const Raw8<float>& r) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, r.w[i] & 0x7fffffffu);
  return m;
}
__device__ __forceinline__ uint32_t amax_pairs(const uint32_t (&w)[4]) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) m = __vmaxu2(m, w[i] & 0x7fff7fffu);
  return max(m >> 16, m & 0xffffu);
}
__device__ __forceinline__ uint32_t amax_bits8(const Raw8<__nv_bfloat16>& r) { return amax_pairs(r.w) << 16; }
__device__ __forceinline__ uint32_t amax_bits8(const Raw8<__half>& r) {
  return __float_as_uint(__half2float(__ushort_as_half(static_cast<unsigned short>(amax_pairs(r.w)))));
}
// The block's e8m0 byte: floor(log2(amax)) - emax + 127, held to 0 or above; 255 (NaN) where amax is not finite. The
// exponent field of amax is floor(log2) + 127 for a normal number, and both subnormals and zero end at byte 0.
template <int FMT>
__device__ __forceinline__ uint32_t scale_byte(uint32_t amax_bits) {
  constexpr int emax = FMT == KO_MXFP4 ? 2 : 8;
  const int e = static_cast<int>(amax_bits >> 23);
  return e == 255 ? 255u : static_cast<uint32_t>(max(e - emax, 0));
}
// 2^(127 - byte), the exact reciprocal of the scale (byte <= 252 where it is not NaN); 0 for a NaN scale, whose block
// holds zero codes.
__device__ __forceinline__ float scale_inverse(uint32_t byte) {
  return byte == 255u ? 0.f : __uint_as_float((254u - byte) << 23);
}
// 2^(byte - 127); byte 0 is the subnormal 2^-127, byte 255 NaN.
__device__ __forceinline__ float scale_value(uint32_t byte) {
  return byte == 0u ? __uint_as_float(0x00400000u) : byte == 255u ? __uint_as_float(0x7fc00000u)
                                                                  : __uint_as_float(byte << 23);
}

// Eight scaled values to e2m1 codes (element 0 in the lowest nibble), to nearest even, saturating at 6.
__device__ __forceinline__ uint32_t pack_e2m1x8(const float (&v)[8], float inv) {
  uint32_t r;
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
      "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
      : "=r"(r)
      : "f"(v[0] * inv), "f"(v[1] * inv), "f"(v[2] * inv), "f"(v[3] * inv), "f"(v[4] * inv), "f"(v[5] * inv),
        "f"(v[6] * inv), "f"(v[7] * inv));
  return r;
}
// Eight scaled values to e4m3 codes, to nearest even, saturating at 448.
__device__ __forceinline__ uint2 pack_e4m3x8(const float (&v)[8], float inv) {
  uint2 r;
  asm("{\n\t.reg .b16 h0, h1, h2, h3;\n\t"
      "cvt.rn.satfinite.e4m3x2.f32 h0, %3, %2;\n\t"
      "cvt.rn.satfinite.e4m3x2.f32 h1, %5, %4;\n\t"
      "cvt.rn.satfinite.e4m3x2.f32 h2, %7, %6;\n\t"
      "cvt.rn.satfinite.e4m3x2.f32 h3, %9, %8;\n\t"
      "mov.b32 %0, {h0, h1};\n\tmov.b32 %1, {h2, h3};\n\t}"
      : "=r"(r.x), "=r"(r.y)
      : "f"(v[0] * inv), "f"(v[1] * inv), "f"(v[2] * inv), "f"(v[3] * inv), "f"(v[4] * inv), "f"(v[5] * inv),
        "f"(v[6] * inv), "f"(v[7] * inv));
  return r;
}
// Eight e2m1 codes as fp32 (exact in fp16 on the way). The bytes are taken apart inside the asm, from a whole 32-bit word:
// fed from an 8-bit load, the conversion came out as zeros (CUDA 12.9).
__device__ __forceinline__ void unpack_e2m1x8(uint32_t w, float (&v)[8]) {
  uint32_t h[4];
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\tmov.b32 {b0, b1, b2, b3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\n\tcvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, b2;\n\tcvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(w));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<__half2*>(&h[i]));
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}
// Two e4m3 codes of a half word as fp32.
__device__ __forceinline__ float2 unpack_e4m3x2(uint32_t half_word) {
  uint32_t h;
  asm("{\n\t.reg .b16 b;\n\tcvt.u16.u32 b, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, b;\n\t}" : "=r"(h) : "r"(half_word));
  return __half22float2(*reinterpret_cast<__half2*>(&h));
}

// Byte offset of the scale word (the four scales of 128 elements) of (row, k tile).
__device__ __forceinline__ int64_t scale_word_offset(int64_t row, int64_t ktile, int64_t ktiles) {
  const int r = static_cast<int>(row & 127);
  return ((row >> 7) * ktiles + ktile) * 512 + (r & 31) * 16 + (r >> 5) * 4;
}

// 32 / L elements of a block at `p`, of which `left` (any integer) lie before the end of the row; the others are zero.
template <typename T, bool VEC, int G>
__device__ __forceinline__ void load_block(const T* p, int left, Raw8<T> (&r)[G]) {
#pragma unroll
  for (int g = 0; g < G; ++g) r[g] = load8<T, VEC>(p + g * 8, left - g * 8);
}
// Their codes (16 / L bytes in mxfp4, 32 / L in mxfp8) and the block's scale byte, the block being shared by L neighbouring
// lanes that call this together.
template <typename T, int FMT, int L>
__device__ __forceinline__ uint32_t quantize_block(const Raw8<T> (&r)[4 / L], uint32_t (&code)[(FMT == KO_MXFP4 ? 4 : 8) / L]) {
  constexpr int G = 4 / L;  // groups of eight
  uint32_t m = 0;
#pragma unroll
  for (int g = 0; g < G; ++g) m = max(m, amax_bits8(r[g]));
#pragma unroll
  for (int s = 1; s < L; s <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, s));
  const uint32_t byte = scale_byte<FMT>(m);
  const float inv = scale_inverse(byte);
#pragma unroll
  for (int g = 0; g < G; ++g) {
    float v[8];
    widen8(r[g], v);
    if constexpr (FMT == KO_MXFP4) {
      code[g] = pack_e2m1x8(v, inv);
    } else {
      const uint2 c = pack_e4m3x8(v, inv);
      code[2 * g] = c.x;
      code[2 * g + 1] = c.y;
    }
  }
  // a NaN or an infinity times the zero inverse is NaN, which would convert to the largest code: such blocks are cleared
  if (byte == 255u) {
#pragma unroll
    for (int i = 0; i < (FMT == KO_MXFP4 ? 1 : 2) * G; ++i) code[i] = 0u;
  }
  return byte;
}

// Writes the codes of a lane's eight values and, from one lane in sixteen, the scale word of their 128 elements. A group
// of sixteen lanes that calls this together holds one row's elements [128 kt, 128 kt + 128) in order; `mask` names them, m
// is the largest magnitude of the lane's own values, `code` the address of their codes.
template <int FMT>
__device__ __forceinline__ void quantize_group(const float (&v)[8], uint32_t m, uint32_t mask, uint8_t* code,
                                               uint8_t* scale_word) {
  const int lane16 = threadIdx.x & 15;
  m = max(m, __shfl_xor_sync(mask, m, 1));
  m = max(m, __shfl_xor_sync(mask, m, 2));
  const uint32_t byte = scale_byte<FMT>(m);
  const float inv = scale_inverse(byte);
  if constexpr (FMT == KO_MXFP4) {
    const uint32_t c = pack_e2m1x8(v, inv);
    *reinterpret_cast<uint32_t*>(code) = byte == 255u ? 0u : c;
  } else {
    uint2 c = pack_e4m3x8(v, inv);
    if (byte == 255u) c = make_uint2(0u, 0u);
    *reinterpret_cast<uint2*>(code) = c;
  }
  // bytes of lanes 0, 4, 8, 12 into lane 0's word
  const uint32_t pair = byte | (__shfl_down_sync(mask, byte, 4, 16) << 8);
  const uint32_t word = pair | (__shfl_down_sync(mask, pair, 8, 16) << 16);
  if (lane16 == 0) *reinterpret_cast<uint32_t*>(scale_word) = word;
}

#endif  // __CUDACC__

}  // namespace komx
