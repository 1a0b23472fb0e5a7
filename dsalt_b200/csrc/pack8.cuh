// The 8-bit form of activations (see pack8.cu) and conversions of 16-bit pairs.
#pragma once

#include <type_traits>

#include "common.cuh"

namespace dsalt {

constexpr int GROUP8 = 32;  // values that share a scale

template <typename T>
__device__ __forceinline__ float to_float(T v);
template <>
__device__ __forceinline__ float to_float(float v) { return v; }
template <>
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_float(float v) { return __float2half_rn(v); }

// two 16-bit values of a register as fp32, and back (round to nearest even)
template <typename T>
__device__ __forceinline__ void widen2(uint32_t u, float& lo, float& hi) {
  if constexpr (sizeof(T) == 2) {
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      lo = __uint_as_float(u << 16);
      hi = __uint_as_float(u & 0xffff0000u);
    } else {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u));
      lo = f.x;
      hi = f.y;
    }
  }
}
template <typename T>
__device__ __forceinline__ uint32_t narrow2(float lo, float hi) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) return pack_bf16x2(lo, hi);
  else return pack_f16x2(lo, hi);
}

// the scale byte of a group whose largest magnitude has the bits `top`
__device__ __forceinline__ uint32_t scale_byte(uint32_t top) {
  const int e = (int)(top >> 23);
  return e == 255 ? 255u : (uint32_t)max(e - 6, 1);
}
// 2^(127 - s), of which the codes are formed; 0 for a group that is not finite (its codes are 0)
__device__ __forceinline__ float inverse_scale(uint32_t s) { return __uint_as_float(s == 255 ? 0u : (254u - s) << 23); }
// 2^(s - 127), or NaN
__device__ __forceinline__ float scale_of(uint32_t s) { return __uint_as_float(s == 255 ? 0x7fffffffu : s << 23); }

// 1.5 * 2^23 + the nearest whole number: its low byte is the code. The product is exact, so the
// sum is rounded once; a NaN (of a group with s = 255) is turned into 0 by the bounds.
__device__ __forceinline__ uint32_t code_bits(float x, float inv) {
  constexpr float C = 12582912.f;
  return __float_as_uint(fminf(fmaxf(fmaf(x, inv, C), C - 127.f), C + 127.f));
}
__device__ __forceinline__ int code_of(float x, uint32_t s) {
  return s == 255 ? 0 : (int)(int8_t)(code_bits(x, inverse_scale(s)) & 0xffu);
}
template <int N>
__device__ __forceinline__ void pack_codes(const float (&f)[N], uint32_t s, uint32_t (&w)[N / 4]) {
  const float inv = inverse_scale(s);
#pragma unroll
  for (int i = 0; i < N / 4; ++i) {
    const uint32_t a = __byte_perm(code_bits(f[4 * i], inv), code_bits(f[4 * i + 1], inv), 0x0040);
    const uint32_t b = __byte_perm(code_bits(f[4 * i + 2], inv), code_bits(f[4 * i + 3], inv), 0x0040);
    w[i] = s == 255 ? 0u : __byte_perm(a, b, 0x5410);
  }
}
template <int N>
__device__ __forceinline__ void unpack_codes(const uint32_t (&w)[N / 4], float scale, float (&f)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) f[i] = (float)(int8_t)(w[i / 4] >> (8 * (i % 4))) * scale;
}

int launch_pack8(const void* x, int dtype, int64_t rows, int64_t cols, int64_t x_stride, int8_t* codes, uint8_t* exps,
                 cudaStream_t stream);
int launch_unpack8(const int8_t* codes, const uint8_t* exps, int64_t rows, int64_t cols, void* out, int dtype,
                   cudaStream_t stream);

}  // namespace dsalt
