// What the two forms of the norm and rotation of queries and keys share (heads.cu: runs of channels; heads_any.cu:
// single channels): angles, a block's constants, the sum over the blocks' partial gradients.
//
// Angles: a position times the pair's frequency in quarter turns in 64 bits, less the nearest whole
// number of them (exact), then sine and cosine in 32 bits of at most an eighth of a turn: a position of 2^20
// keeps the digits that a 32-bit product would lose.
#pragma once

#include "common.cuh"
#include "kernels.h"

namespace ffb {
namespace heads {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMostBlocks = 148 * 4;  // rows of partial gradients of q's, and as many of k's

// Cosine and sine of an angle of at most an eighth of a turn, r quarter turns (|r| <= 1/2): polynomials in r^2
// through Chebyshev's nodes. With coefficients in 32 bits they are off by 0.12 (cosine) and 0.4 (sine) steps of 2^-24; with
// the roundings of r and of their evaluation by 1.3 and 1.7 (20 million angles).
__device__ __forceinline__ float2 eighth_turn(float r) {
  const float t = r * r;
  const float s = r * fmaf(fmaf(fmaf(-0.0046021491289f, t, 0.0796802192926f), t, -0.6459634900093f), t, 1.5707963705063f);
  const float c = fmaf(fmaf(fmaf(fmaf(0.0009036280680f, t, -0.0208600703627f), t, 0.2536692023277f), t, -1.2337005138397f), t, 1.0f);
  return make_float2(c, s);
}

// cosine and sine of the angle of `quarters` quarter turns
__device__ __forceinline__ float2 turn_of(double quarters, uint32_t inverse_sign) {
  // the nearest whole number: 1.5 2^52 has a last place of 1, so the sum rounds to it, and its lowest bits are the
  // number's. (Past 2^51 neighbouring doubles are half a quarter turn and more apart.)
  double whole = quarters + 6755399441055744.0;
  int k = __double2loint(whole);
  whole -= 6755399441055744.0;
  if (!(fabs(quarters) < 2251799813685248.0)) {
    whole = rint(quarters);
    k = static_cast<int>(whole - 4.0 * rint(0.25 * whole));
  }
  const float2 t = eighth_turn(static_cast<float>(quarters - whole));
  // k quarter turns more
  const float cos = k & 1 ? t.y : t.x, sin = k & 1 ? t.x : t.y;
  return make_float2(__uint_as_float(__float_as_uint(cos) ^ (((k + 1) & 2) << 30)),
                     __uint_as_float(__float_as_uint(sin) ^ ((k & 2) << 30) ^ inverse_sign));
}

// the position at element `i`
__device__ __forceinline__ double position_at(const RotaryParams& r, int64_t i) {
  if (r.type == kPositionI64) return static_cast<double>(static_cast<const int64_t*>(r.positions)[i]);
  if (r.type == kPositionI32) return static_cast<double>(static_cast<const int32_t*>(r.positions)[i]);
  return static_cast<double>(static_cast<const float*>(r.positions)[i]);
}

// What a block reads again for every token, from its start on in shared memory, so that the first token waits for
// one load's time and not for several one after the other: the pairs' frequencies and axes, q's and k's weights.
struct Constants {
  double* quarters;  // [slots]; NaN where a pair's axis is not there
  int* axes;
  float* weights;  // [2][channels, to a multiple of 4]
  __host__ __device__ static int padded(int channels) { return (channels + 3) / 4 * 4; }
  __host__ __device__ static int bytes(int slots, int channels) { return slots * 12 + padded(channels) * 8; }
  __device__ __forceinline__ Constants(const HeadsParams& p, int slots, uint8_t* smem) {
    quarters = reinterpret_cast<double*>(smem);
    weights = reinterpret_cast<float*>(quarters + slots);
    axes = reinterpret_cast<int*>(weights + 2 * padded(p.channels));
    const RotaryParams& r = p.rotary;
    for (int j = threadIdx.x; j < r.pairs; j += kThreads) {
      const int axis = r.pair_axes[j];
      const double q = r.quarters[j];
      const bool there = axis >= 0 && axis < r.axes;
      quarters[j] = there ? q : __longlong_as_double(0x7FF8000000000000LL);
      axes[j] = there ? axis : 0;
    }
    for (int c = threadIdx.x; c < 2 * padded(p.channels); c += kThreads) {
      const int which = c >= padded(p.channels), i = c - which * padded(p.channels);
      weights[c] = p.weight[which] != nullptr && i < p.channels ? p.weight[which][i] : 1.f;
    }
  }
  __device__ __forceinline__ const float* weight(const HeadsParams& p, int which) const { return weights + which * padded(p.channels); }
};

// The weights' gradients from the blocks' partial sums (q's rows, then k's), in a fixed order.
int reduce(const float* part, const HeadsParams& p, int blocks, cudaStream_t stream);

// single channels, for heads that are not whole runs (heads_any.cu)
template <typename T>
int forward_any(const HeadsParams& p, cudaStream_t stream);
template <typename T>
int backward_any(const HeadsParams& p, float* part, cudaStream_t stream);

}  // namespace heads
}  // namespace ffb
