// The 8-bit form activations are kept in for a backward pass: a row's channels in blocks of 32,
// e4m3 codes and one power-of-two scale (a biased exponent byte, 2^(byte - 127)) a block.
//
// The scale is the smallest power of two that brings the block's largest finite magnitude A to at
// most 448, e4m3's largest: with A = m 2^E, m in [1, 2), that is 2^(E - 8), or 2^(E - 7) where m >
// 1.75. (Scaling by 2^(E - 8) always would cut values between 448 and 512 down to 448, an error of up
// to 1/8 where rounding alone makes at most 1/16.) Scaling by a power of two is exact, so a code
// depends on its block's values alone: no order of summation and no rounding before it can move it
// over a border. Values that are not finite become the NaN code and take no part in A.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

namespace ffb {

constexpr int kMxBlock = 32;

// |x| where x is finite, else 0 (a NaN compares false)
__device__ __forceinline__ float mx_magnitude(float x) {
  const float a = fabsf(x);
  return a <= 3.402823466e38f ? a : 0.f;
}

// The scale byte of a block from its largest finite magnitude: the biased exponent less 8, one more
// where the mantissa is above 1.75 (adding 0x1FFFFF carries into the exponent exactly then).
__device__ __forceinline__ uint32_t mx_scale_byte(float largest) {
  const int e = static_cast<int>((__float_as_uint(largest) + 0x1FFFFFu) >> 23) - 8;
  return static_cast<uint32_t>(e > 0 ? e : 0);
}

// 2^(byte - 127) and its inverse (byte <= 247 for every scale mx_scale_byte gives)
__device__ __forceinline__ float mx_scale(uint32_t byte) {
  return __uint_as_float(byte != 0 ? byte << 23 : 0x00400000u);
}
__device__ __forceinline__ float mx_inverse_scale(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }

// two values, already scaled, to e4m3 (round to nearest even): lo in the low byte
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
// x * inv, or NaN where x is not finite (the conversion above would make 448 of an infinity)
__device__ __forceinline__ float mx_scaled(float x, float inv) {
  return fabsf(x) <= 3.402823466e38f ? x * inv : __uint_as_float(0x7FFFFFFFu);
}

// two codes to fp32 (exact)
__device__ __forceinline__ float2 e4m3x2_value(uint32_t pair) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(static_cast<uint16_t>(pair)));
  return __half22float2(*reinterpret_cast<__half2*>(&h));
}

// the largest magnitude over the `LANES` consecutive lanes that share a block
template <int LANES>
__device__ __forceinline__ float mx_block_max(float a) {
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) a = fmaxf(a, __shfl_xor_sync(0xFFFFFFFFu, a, o));
  return a;
}

// ------------------------------------------------------------------ vectors of VEC elements
template <int VEC>
struct MxCodes;  // VEC code bytes as one machine word
template <>
struct MxCodes<8> { using type = uint2; };
template <>
struct MxCodes<4> { using type = uint32_t; };
template <>
struct MxCodes<1> { using type = uint8_t; };

template <int VEC>
__device__ __forceinline__ typename MxCodes<VEC>::type mx_encode(const float (&f)[VEC], float inv) {
  if constexpr (VEC == 1) {
    const float v = mx_scaled(f[0], inv);
    return static_cast<uint8_t>(e4m3x2(v, 0.f));
  } else {
    uint32_t w[VEC / 4];
#pragma unroll
    for (int i = 0; i < VEC / 4; ++i)
      w[i] = e4m3x2(mx_scaled(f[4 * i], inv), mx_scaled(f[4 * i + 1], inv)) |
             (e4m3x2(mx_scaled(f[4 * i + 2], inv), mx_scaled(f[4 * i + 3], inv)) << 16);
    if constexpr (VEC == 8)
      return make_uint2(w[0], w[1]);
    else
      return w[0];
  }
}

template <int VEC>
__device__ __forceinline__ void mx_decode(typename MxCodes<VEC>::type codes, float scale, float (&f)[VEC]) {
  if constexpr (VEC == 1) {
    f[0] = e4m3x2_value(codes).x * scale;
  } else {
    uint32_t w[VEC / 4];
    if constexpr (VEC == 8) {
      w[0] = codes.x;
      w[1] = codes.y;
    } else {
      w[0] = codes;
    }
#pragma unroll
    for (int i = 0; i < VEC / 4; ++i) {
      const float2 lo = e4m3x2_value(w[i] & 0xFFFFu), hi = e4m3x2_value(w[i] >> 16);
      f[4 * i] = lo.x * scale;
      f[4 * i + 1] = lo.y * scale;
      f[4 * i + 2] = hi.x * scale;
      f[4 * i + 3] = hi.y * scale;
    }
  }
}

// VEC elements of type T to and from fp32: VEC is a 16-byte load's worth (8 bf16, 4 fp32), or 1
template <typename T, int VEC>
__device__ __forceinline__ void load_vec(const T* p, float (&f)[VEC]) {
  if constexpr (VEC == 1) {
    f[0] = static_cast<float>(*p);
  } else if constexpr (sizeof(T) == 4) {
    const float4 v = *reinterpret_cast<const float4*>(p);
    f[0] = v.x;
    f[1] = v.y;
    f[2] = v.z;
    f[3] = v.w;
  } else {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
  }
}

template <typename T, int VEC>
__device__ __forceinline__ void store_vec(T* p, const float (&f)[VEC]) {
  if constexpr (VEC == 1) {
    *p = static_cast<T>(f[0]);  // round to nearest even
  } else if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
  } else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

}  // namespace ffb
