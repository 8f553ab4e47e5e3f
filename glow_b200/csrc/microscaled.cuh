// The microscaled 4-bit format on the device, and float operands of several types.
#pragma once
#include <cuda_bf16.h>

#include <type_traits>

#include "common.cuh"

namespace glowb200 {

constexpr int kMxBlock = 32;  // elements that share a scale
inline int64_t mx_blocks(int64_t cols) { return (cols + kMxBlock - 1) / kMxBlock; }
inline int64_t mx_pitch(int64_t cols) { return 16 * mx_blocks(cols); }         // bytes of a packed row
inline int64_t mx_tiles(int64_t cols) { return (mx_blocks(cols) + 3) / 4; }    // scale tiles along a row
inline int64_t mx_row_tiles(int64_t rows) { return (rows + 127) / 128; }

inline bool aligned(const void *p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }
// Whether `n` bytes at p lie beside all of `rows` rows of `m` bytes, `stride` bytes apart, from q on.
inline bool apart(const void *p, size_t n, const void *q, size_t m, size_t rows = 1, size_t stride = 0) {
  const uintptr_t a = reinterpret_cast<uintptr_t>(p), b = reinterpret_cast<uintptr_t>(q);
  if (a < b) return n <= b - a;
  const size_t row = rows > 1 ? (a - b) / stride : 0, at = a - b - row * stride;  // in front of the first byte
  return row >= rows || (at >= m && (row + 1 >= rows || n <= stride - at));
}
inline int float_type_bytes(int type) { return type == GLOWB200_FLOAT32 ? 4 : 2; }
// Calls f with a null pointer of the element type behind GLOWB200_FLOAT32 / FLOAT16 / BFLOAT16.
template <typename F>
int with_float_type(int type, F f) {
  switch (type) {
    case GLOWB200_FLOAT32: return f(static_cast<float *>(nullptr));
    case GLOWB200_FLOAT16: return f(static_cast<__half *>(nullptr));
    case GLOWB200_BFLOAT16: return f(static_cast<__nv_bfloat16 *>(nullptr));
    default: return set_error(GLOWB200_ERR_INVALID_ARGUMENT, "float type %d is not GLOWB200_FLOAT32, _FLOAT16 or _BFLOAT16", type);
  }
}

int run_mx_quantize(const void *in, int in_type, int64_t rows, int64_t cols, int64_t row_stride, uint8_t *data, uint8_t *scales,
                    cudaStream_t s);

#ifdef __CUDACC__
__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ float from_float<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

__device__ __forceinline__ uint32_t pack2(float lo, float hi, __half) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi, __nv_bfloat16) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// Scale byte of a block whose largest magnitude has these fp32 bits (sign bit clear): the biased exponent less two is
// e + 127; infinities and NaNs have exponent 255.  (Magnitudes below 2^-124, subnormal ones too, take the smallest scale.)
__device__ __forceinline__ uint32_t mx_scale_byte(uint32_t top) {
  const uint32_t e = top >> 23;
  return e == 255u ? 255u : e > 2u ? e - 2u : 0u;
}
// 2^-e for a scale byte of 0..252: exact, and so is its product with every element of the block that rounds to a number
// other than 0.
__device__ __forceinline__ float mx_inverse_scale(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }
// The scale itself: 2^-127 is subnormal, 255 a NaN.
__device__ __forceinline__ float mx_scale(uint32_t byte) {
  return __uint_as_float(byte == 0u ? 0x00400000u : byte == 255u ? 0x7FC00000u : byte << 23);
}
// Eight scaled numbers -> eight E2M1 codes, the first in the low bits (nearest, ties to even, saturating).
__device__ __forceinline__ uint32_t mx_codes(const float (&v)[8]) {
  uint32_t r;
  asm("{\n\t.reg .b8 c0, c1, c2, c3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c0, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c2, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c3, %8, %7;\n\t"
      "mov.b32 %0, {c0, c1, c2, c3};\n\t}"
      : "=r"(r)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return r;
}
// Eight neighbours of a row from `x` on, `left` of which are there (the others are zeros).  VEC: x is on a 16-byte boundary.
template <bool VEC, typename T>
struct Eight {
  __align__(16) T w[8];
  __device__ __forceinline__ void load(const T *x, int64_t left) {
    if (VEC && left >= 8) {
#pragma unroll
      for (int k = 0; k < (int)(8 * sizeof(T) / 16); k++) reinterpret_cast<uint4 *>(w)[k] = __ldg(reinterpret_cast<const uint4 *>(x) + k);
    } else {
#pragma unroll
      for (int k = 0; k < 8; k++) w[k] = k < left ? x[k] : from_float<T>(0.0f);
    }
  }
};
// A block of 32 numbers, eight to each of four neighbouring lanes (all 32 lanes take part): the lane's codes and the block's
// scale byte.  Infinities and NaNs: byte 255, codes 0.
template <bool VEC, typename T>
__device__ __forceinline__ uint32_t mx_block(const Eight<VEC, T> &x, uint32_t &byte) {
  uint32_t top = 0;  // the largest magnitude's bits
  float v[8];
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int k = 0; k < 8; k++) {
      v[k] = x.w[k];
      top = max(top, __float_as_uint(v[k]) & 0x7FFFFFFFu);
    }
  } else {  // two at a time: magnitudes are ordered as their bits are
    const uint32_t *w = reinterpret_cast<const uint32_t *>(x.w);
    uint32_t most = __vmaxu2(__vmaxu2(w[0] & 0x7FFF7FFFu, w[1] & 0x7FFF7FFFu), __vmaxu2(w[2] & 0x7FFF7FFFu, w[3] & 0x7FFF7FFFu));
    most = max(most & 0xFFFFu, most >> 16);
    if constexpr (std::is_same_v<T, __half>) top = __float_as_uint(__half2float(__ushort_as_half((unsigned short)most)));
    else top = most << 16;
#pragma unroll
    for (int k = 0; k < 8; k++) v[k] = to_float(x.w[k]);
  }
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
  byte = mx_scale_byte(top);
  const float inverse = mx_inverse_scale(byte == 255u ? 127u : byte);
#pragma unroll
  for (int k = 0; k < 8; k++) v[k] *= inverse;
  return byte == 255u ? 0u : mx_codes(v);
}
// Two codes (a byte) -> their numbers.
__device__ __forceinline__ float2 mx_numbers(uint32_t byte) {
  uint32_t h;
  asm("{\n\t.reg .b8 c, d0, d1, d2;\n\t"
      "mov.b32 {c, d0, d1, d2}, %1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, c;\n\t}"
      : "=r"(h)
      : "r"(byte));
  return __half22float2(*reinterpret_cast<const __half2 *>(&h));
}
#endif

}  // namespace glowb200
