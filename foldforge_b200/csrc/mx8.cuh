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
#include <string.h>

#include "common.cuh"

namespace ffb {

constexpr int kMxBlock = 32;

// The scale byte of a block from the bits of its largest finite magnitude: the biased exponent less 8, one
// more where the mantissa is above 1.75 (adding 0x1FFFFF carries into the exponent exactly then).
__device__ __forceinline__ uint32_t mx_scale_byte(uint32_t largest) {
  const int e = static_cast<int>((largest + 0x1FFFFFu) >> 23) - 8;
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
// two codes to fp32 (exact)
__device__ __forceinline__ float2 e4m3x2_value(uint32_t pair) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(static_cast<uint16_t>(pair)));
  return __half22float2(*reinterpret_cast<__half2*>(&h));
}

// ------------------------------------------------------------------ vectors of VEC elements
// VEC fp32 values of a thread, in pairs on the paired fp32 pipe (or a single one)
template <int VEC>
struct Lanes {
  uint64_t p[VEC / 2];
  __device__ __forceinline__ Lanes() {}
  __device__ __forceinline__ explicit Lanes(float x) {
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) p[i] = f32x2(x, x);
  }
  template <typename F>
  __device__ __forceinline__ Lanes each(F&& f) const {
    Lanes r;
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) {
      float a, b;
      f32x2_split(p[i], a, b);
      a = f(a);
      b = f(b);
      r.p[i] = f32x2(a, b);
    }
    return r;
  }
  // f(this value, the other's)
  template <typename F>
  __device__ __forceinline__ Lanes apply(const Lanes& o, F&& f) const {
    Lanes r;
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) {
      float a, b, c, d;
      f32x2_split(p[i], a, b);
      f32x2_split(o.p[i], c, d);
      c = f(a, c);
      d = f(b, d);
      r.p[i] = f32x2(c, d);
    }
    return r;
  }
  __device__ __forceinline__ float sum() const {
    uint64_t t = p[0];
#pragma unroll
    for (int i = 1; i < VEC / 2; ++i) t = add_f32x2(t, p[i]);
    float a, b;
    f32x2_split(t, a, b);
    return a + b;
  }
  // the sum as a tree: equal values add up without rounding
  __device__ __forceinline__ float tree() const {
    uint64_t t[VEC / 2];
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) t[i] = p[i];
#pragma unroll
    for (int n = VEC / 4; n > 0; n /= 2)
#pragma unroll
      for (int i = 0; i < n; ++i) t[i] = add_f32x2(t[i], t[i + n]);
    float a, b;
    f32x2_split(t[0], a, b);
    return a + b;
  }
  // the sum of products with `o`
  __device__ __forceinline__ float dot(const Lanes& o) const {
    uint64_t t = mul_f32x2(p[0], o.p[0]);
#pragma unroll
    for (int i = 1; i < VEC / 2; ++i) t = fma_f32x2(p[i], o.p[i], t);
    float a, b;
    f32x2_split(t, a, b);
    return a + b;
  }
  __device__ __forceinline__ float get(int j) const {
    float a, b;
    f32x2_split(p[j / 2], a, b);
    return j & 1 ? b : a;
  }
};
template <>
struct Lanes<1> {
  float f;
  __device__ __forceinline__ Lanes() {}
  __device__ __forceinline__ explicit Lanes(float x) : f(x) {}
  template <typename F>
  __device__ __forceinline__ Lanes each(F&& g) const {
    return Lanes(g(f));
  }
  template <typename F>
  __device__ __forceinline__ Lanes apply(const Lanes& o, F&& g) const {
    return Lanes(g(f, o.f));
  }
  __device__ __forceinline__ float sum() const { return f; }
  __device__ __forceinline__ float tree() const { return f; }
  __device__ __forceinline__ float dot(const Lanes& o) const { return f * o.f; }
  __device__ __forceinline__ float get(int) const { return f; }
};
template <int VEC>
__device__ __forceinline__ Lanes<VEC> operator+(const Lanes<VEC>& a, const Lanes<VEC>& b) {
  Lanes<VEC> r;
  if constexpr (VEC == 1) {
    r.f = a.f + b.f;
  } else {
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) r.p[i] = add_f32x2(a.p[i], b.p[i]);
  }
  return r;
}
template <int VEC>
__device__ __forceinline__ Lanes<VEC> operator*(const Lanes<VEC>& a, const Lanes<VEC>& b) {
  Lanes<VEC> r;
  if constexpr (VEC == 1) {
    r.f = a.f * b.f;
  } else {
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) r.p[i] = mul_f32x2(a.p[i], b.p[i]);
  }
  return r;
}
template <int VEC>
__device__ __forceinline__ Lanes<VEC> fma(const Lanes<VEC>& a, const Lanes<VEC>& b, const Lanes<VEC>& c) {
  Lanes<VEC> r;
  if constexpr (VEC == 1) {
    r.f = fmaf(a.f, b.f, c.f);
  } else {
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) r.p[i] = fma_f32x2(a.p[i], b.p[i], c.p[i]);
  }
  return r;
}
// VEC values of a weight vector (16-byte aligned where VEC > 1)
template <int VEC>
__device__ __forceinline__ Lanes<VEC> load_weight(const float* p) {
  Lanes<VEC> r;
  if constexpr (VEC == 1) {
    r.f = __ldg(p);
  } else {
#pragma unroll
    for (int i = 0; i < VEC / 4; ++i) {
      const float4 v = __ldg(reinterpret_cast<const float4*>(p) + i);
      r.p[2 * i] = f32x2(v.x, v.y);
      r.p[2 * i + 1] = f32x2(v.z, v.w);
    }
  }
  return r;
}

template <int VEC>
struct MxCodes;  // VEC code bytes as one machine word
template <>
struct MxCodes<8> { using type = uint2; };
template <>
struct MxCodes<4> { using type = uint32_t; };
template <>
struct MxCodes<1> { using type = uint8_t; };

template <int VEC>
__device__ __forceinline__ typename MxCodes<VEC>::type mx_encode(const Lanes<VEC>& v) {
  typename MxCodes<VEC>::type out;
  if constexpr (VEC == 1) {
    out = static_cast<uint8_t>(e4m3x2(v.f, 0.f));
  } else {
    uint32_t w[VEC / 4];
#pragma unroll
    for (int i = 0; i < VEC / 4; ++i) {
      float a, b, c, d;
      f32x2_split(v.p[2 * i], a, b);
      f32x2_split(v.p[2 * i + 1], c, d);
      w[i] = e4m3x2(a, b) | (e4m3x2(c, d) << 16);
    }
    memcpy(&out, w, sizeof(out));
  }
  return out;
}

// VEC codes as fp32, without their scale (exact)
template <int VEC>
__device__ __forceinline__ Lanes<VEC> mx_codes_value(const typename MxCodes<VEC>::type& codes) {
  Lanes<VEC> v;
  if constexpr (VEC == 1) {
    v.f = e4m3x2_value(codes).x;
  } else {
    uint32_t w[VEC / 4];
    memcpy(w, &codes, sizeof(codes));
#pragma unroll
    for (int i = 0; i < VEC / 4; ++i) {
      const float2 lo = e4m3x2_value(w[i] & 0xFFFFu), hi = e4m3x2_value(w[i] >> 16);
      v.p[2 * i] = f32x2(lo.x, lo.y);
      v.p[2 * i + 1] = f32x2(hi.x, hi.y);
    }
  }
  return v;
}

// Eight codes times their scale as bf16, exactly (e4m3's 4 significant bits fit bf16's 8; only below 2^-126
// may the result round). A code's exponent and mantissa, moved to bf16's fields as they are, stand for the
// value times 2^-120 (biases 7 and 127), subnormal codes included; a multiplication by 2^(byte - 7) makes
// the value of it. Integer and paired bf16 operations only: the conversion instruction runs at a fraction
// of their rate.
__device__ __forceinline__ uint4 mx_decode_bf16(uint2 codes, uint32_t byte) {
  const uint32_t c[2] = {codes.x, codes.y};
  uint32_t w[4];
  const uint32_t scale = (byte + 120u) * 0x00800080u;  // 2^(byte - 7) twice, for bytes up to 134
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t t = __byte_perm(c[i / 2], 0, i & 1 ? 0x3424 : 0x1404);  // each code in the high byte of its half
    w[i] = (t & 0x80008000u) | ((t >> 4) & 0x07F007F0u);
  }
  // NaN codes (all seven bits set), or a scale of more than 2^7, whose product with 2^120 is past bf16's range
  const uint32_t n0 = ((c[0] & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u, n1 = ((c[1] & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u;
  if ((n0 | n1) != 0 || byte > 134u) {
    const uint32_t s16 = byte != 0 ? byte << 7 : 0x0040u;  // 2^(byte - 127) in bf16
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(w[i]) : "r"(w[i]), "r"(0x7B807B80u));  // 2^120
      asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(w[i]) : "r"(w[i]), "r"(s16 | (s16 << 16)));
      const uint32_t n = (i < 2 ? n0 : n1) >> (16 * (i & 1));
      if (n & 0x80u) w[i] |= 0x00007FFFu;
      if (n & 0x8000u) w[i] |= 0x7FFF0000u;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(w[i]) : "r"(w[i]), "r"(scale));
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// VEC elements of type T as they lie in memory: whole 16-byte words, or one element. Kernels hold rows in
// this form (bf16 in half the registers of fp32) and widen on use.
template <int WORDS>
struct Words {
  uint4 w[WORDS];
};
template <typename T, int VEC>
struct Raw {
  using type = Words<VEC * sizeof(T) / 16>;
};
template <typename T>
struct Raw<T, 1> {
  using type = T;
};

// a load of data that is read once (kept out of the way of what is read again)
template <typename T, int VEC>
__device__ __forceinline__ typename Raw<T, VEC>::type load_raw(const T* p) {
  if constexpr (VEC == 1) {
    return *p;
  } else {
    typename Raw<T, VEC>::type v;
#pragma unroll
    for (int i = 0; i < VEC * static_cast<int>(sizeof(T)) / 16; ++i) v.w[i] = __ldcs(reinterpret_cast<const uint4*>(p) + i);
    return v;
  }
}

// the same from shared memory
template <typename T, int VEC>
__device__ __forceinline__ typename Raw<T, VEC>::type shared_raw(const T* p) {
  return *reinterpret_cast<const typename Raw<T, VEC>::type*>(p);
}

template <typename T, int VEC>
__device__ __forceinline__ typename Raw<T, VEC>::type zero_raw() {
  if constexpr (VEC == 1) {
    return static_cast<T>(0.f);
  } else {
    typename Raw<T, VEC>::type v;
#pragma unroll
    for (int i = 0; i < VEC * static_cast<int>(sizeof(T)) / 16; ++i) v.w[i] = make_uint4(0, 0, 0, 0);
    return v;
  }
}

template <typename T, int VEC>
__device__ __forceinline__ Lanes<VEC> widen(const typename Raw<T, VEC>::type& v) {
  Lanes<VEC> f;
  if constexpr (VEC == 1) {
    f.f = static_cast<float>(v);
  } else {
#pragma unroll
    for (int i = 0; i < VEC * static_cast<int>(sizeof(T)) / 16; ++i) {
      const uint32_t w[4] = {v.w[i].x, v.w[i].y, v.w[i].z, v.w[i].w};
      if constexpr (sizeof(T) == 4) {
        f.p[2 * i] = f32x2(__uint_as_float(w[0]), __uint_as_float(w[1]));
        f.p[2 * i + 1] = f32x2(__uint_as_float(w[2]), __uint_as_float(w[3]));
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) f.p[4 * i + k] = f32x2(bf16_lo(w[k]), bf16_hi(w[k]));
      }
    }
  }
  return f;
}

template <typename T, int VEC>
__device__ __forceinline__ void store_lanes(T* p, const Lanes<VEC>& f) {
  if constexpr (VEC == 1) {
    *p = static_cast<T>(f.f);  // round to nearest even
  } else {
#pragma unroll
    for (int i = 0; i < VEC * static_cast<int>(sizeof(T)) / 16; ++i) {
      uint32_t w[4];
      if constexpr (sizeof(T) == 4) {
        memcpy(w, &f.p[2 * i], 16);
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          float lo, hi;
          f32x2_split(f.p[4 * i + k], lo, hi);
          w[k] = pack_bf16(lo, hi);
        }
      }
      __stcs(reinterpret_cast<uint4*>(p) + i, make_uint4(w[0], w[1], w[2], w[3]));
    }
  }
}

__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("max.u16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}

// The bits (fp32) of the largest magnitude among VEC elements: magnitudes order as their bits do, an
// infinity or a NaN above every finite one. bf16 pairs are compared two at a time.
template <typename T, int VEC>
__device__ __forceinline__ uint32_t max_magnitude(const typename Raw<T, VEC>::type& v) {
  if constexpr (VEC == 1) {
    return __float_as_uint(static_cast<float>(v)) & 0x7FFFFFFFu;
  } else {
    constexpr uint32_t mask = sizeof(T) == 4 ? 0x7FFFFFFFu : 0x7FFF7FFFu;
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < VEC * static_cast<int>(sizeof(T)) / 16; ++i) {
      const uint32_t a = v.w[i].x & mask, b = v.w[i].y & mask, c = v.w[i].z & mask, d = v.w[i].w & mask;
      if constexpr (sizeof(T) == 4)
        m = max(m, max(max(a, b), max(c, d)));
      else
        m = max_u16x2(m, max_u16x2(max_u16x2(a, b), max_u16x2(c, d)));
    }
    return sizeof(T) == 4 ? m : max(m << 16, m & 0xFFFF0000u);
  }
}

// the largest of the lanes that share a block (a whole warp for single elements)
template <int VEC>
__device__ __forceinline__ uint32_t mx_lanes_max(uint32_t m) {
  if constexpr (VEC == 1) return __reduce_max_sync(0xFFFFFFFFu, m);
#pragma unroll
  for (int o = kMxBlock / VEC / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
  return m;
}

// The codes of N vectors of VEC elements of a thread, and the scale byte of each one's block, whose 32
// channels lie in 32 / VEC consecutive lanes. All of a warp's threads call this together. `f` holds the
// widened elements.
template <typename T, int VEC, int N>
__device__ __forceinline__ void mx_quantise(const typename Raw<T, VEC>::type (&v)[N], const Lanes<VEC> (&f)[N],
                                            typename MxCodes<VEC>::type (&codes)[N], uint32_t (&byte)[N]) {
  constexpr uint32_t kInfinity = 0x7F800000u;
  uint32_t m[N], top = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    m[i] = mx_lanes_max<VEC>(max_magnitude<T, VEC>(v[i]));
    top = max(top, m[i]);
  }
  if (__any_sync(0xFFFFFFFFu, top >= kInfinity)) {
    // rare: somewhere in the warp's blocks a value is not finite. It becomes NaN (the conversion to e4m3
    // would make 448 of an infinity) and the scale is that of the others.
#pragma unroll
    for (int i = 0; i < N; ++i) {
      uint32_t largest = 0;
      f[i].each([&](float x) {
        const uint32_t a = __float_as_uint(x) & 0x7FFFFFFFu;
        largest = max(largest, a < kInfinity ? a : 0u);
        return x;
      });
      byte[i] = mx_scale_byte(mx_lanes_max<VEC>(largest));
      const float inv = mx_inverse_scale(byte[i]);
      codes[i] = mx_encode<VEC>(f[i].each([&](float x) {
        return (__float_as_uint(x) & 0x7FFFFFFFu) < kInfinity ? x * inv : __uint_as_float(0x7FFFFFFFu);
      }));
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    byte[i] = mx_scale_byte(m[i]);
    codes[i] = mx_encode<VEC>(f[i] * Lanes<VEC>(mx_inverse_scale(byte[i])));
  }
}

}  // namespace ffb
