// Queries and keys of each head before an attention: divided by their root mean square, scaled by a weight,
// turned in pairs by their positions' angles, and the backward pass; the rotation alone as well.
//
// A warp takes a token's heads, a team of lanes a head: a lane holds the same pairs of channels of every
// head that comes to its team. So the warp finds the token's cosines and sines once for all heads (into
// shared memory, each pair by one lane), folds the weight into them, and a head costs its loads, one sum over
// the team and two multiply-adds a channel. In the backward pass a lane also adds up the weight's gradient of
// its channels over all heads and tokens that it meets.
//
// Angles: a position times the pair's frequency in quarter turns in 64 bits, less the nearest whole
// number of them (exact), then sine and cosine in 32 bits of at most an eighth of a turn: a position of 2^20
// keeps the digits that a 32-bit product would lose.
#include <string.h>

#include <type_traits>

#include "abi_util.h"
#include "common.cuh"
#include "kernels.h"
#include "launch.cuh"
#include "mx8.cuh"

namespace ffb {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;

// cosine and sine of pair `j`'s angle at a token
__device__ __forceinline__ float2 turn_of(const RotaryParams& r, int64_t at, int j) {
  const int axis = r.pair_axes[j];
  if (axis < 0 || axis >= r.axes) return make_float2(__int_as_float(0x7FFFFFFF), __int_as_float(0x7FFFFFFF));
  const int64_t i = at + axis * r.axis;
  double place;
  if (r.type == kPositionI64)
    place = static_cast<double>(static_cast<const int64_t*>(r.positions)[i]);
  else if (r.type == kPositionI32)
    place = static_cast<double>(static_cast<const int32_t*>(r.positions)[i]);
  else
    place = static_cast<double>(static_cast<const float*>(r.positions)[i]);
  const double quarters = place * r.quarters[j];
  const double whole = rint(quarters);
  float s, c;
  sincospif(0.5f * static_cast<float>(quarters - whole), &s, &c);
  // the whole quarter turns, modulo 4
  const int k = static_cast<int>(whole - 4.0 * rint(0.25 * whole)) & 3;
  const float cos = k == 0 ? c : k == 1 ? -s : k == 2 ? -c : s;
  const float sin = k == 0 ? s : k == 1 ? c : k == 2 ? -s : -c;
  return make_float2(cos, r.inverse ? -sin : sin);
}

// A token's cosines and sines of `slots` pairs (those past the table's: no turn) to a warp's shared memory.
__device__ __forceinline__ void find_turns(const RotaryParams& r, int64_t at, int slots, float* cosines, float* sines) {
  __syncwarp();
  for (int j = threadIdx.x & 31; j < slots; j += 32) {
    const float2 t = j < r.pairs ? turn_of(r, at, j) : make_float2(1.f, 0.f);
    cosines[j] = t.x;
    sines[j] = t.y;
  }
  __syncwarp();
}

// P elements side by side in memory
template <typename T, int P>
struct Run {
  uint32_t w[P * sizeof(T) / 4];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (sizeof(w) == 8) {
      const uint2 v = __ldcs(reinterpret_cast<const uint2*>(p));
      memcpy(w, &v, 8);
    } else {
#pragma unroll
      for (int i = 0; i < static_cast<int>(sizeof(w)) / 16; ++i) {
        const uint4 v = __ldcs(reinterpret_cast<const uint4*>(p) + i);
        memcpy(w + 4 * i, &v, 16);
      }
    }
  }
  __device__ __forceinline__ void load_again(const T* p) {  // what every token reads
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(w)) / 16; ++i) {
      const uint4 v = __ldg(reinterpret_cast<const uint4*>(p) + i);
      memcpy(w + 4 * i, &v, 16);
    }
  }
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (sizeof(w) == 8) {
      *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    } else {
#pragma unroll
      for (int i = 0; i < static_cast<int>(sizeof(w)) / 16; ++i)
        reinterpret_cast<uint4*>(p)[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
    }
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(w)) / 4; ++i) w[i] = 0;
  }
  __device__ __forceinline__ float get(int i) const {
    if constexpr (sizeof(T) == 4) return __uint_as_float(w[i]);
    return i & 1 ? bf16_hi(w[i / 2]) : bf16_lo(w[i / 2]);
  }
  __device__ __forceinline__ void set_two(int i, float x, float y) {  // elements i (even) and i + 1
    if constexpr (sizeof(T) == 4) {
      w[i] = __float_as_uint(x);
      w[i + 1] = __float_as_uint(y);
    } else {
      w[i / 2] = pack_bf16(x, y);
    }
  }
};
template <typename T>
struct Run<T, 1> {
  T v;
  __device__ __forceinline__ void load(const T* p) { v = *p; }
  __device__ __forceinline__ void load_again(const T* p) { v = __ldg(p); }
  __device__ __forceinline__ void store(T* p) const { *p = v; }
  __device__ __forceinline__ void zero() { v = static_cast<T>(0.f); }
  __device__ __forceinline__ float get(int) const { return static_cast<float>(v); }
};

// A lane's P pairs of a head: their first channels `a` and second channels `b`.
template <int P>
struct Pairs {
  Lanes<P> a, b;
};

// Where a lane's P pairs lie: runs of P channels at `a` and `b`, which are the pairs' first and second channels,
// or with INTER two halves of a run in which both take turns. P = 1: single channels anywhere.
template <int P>
struct Spot {
  int a, b;    // element offsets in a head
  int turned;  // how many of the pairs are turned: the first ones
  bool has_a, has_b;
};
template <int P, bool INTER>
__device__ __forceinline__ Spot<P> spot_of(const RotaryParams& r, int chunk, int channels) {
  Spot<P> s;
  const int first = chunk * P, turned = r.pairs - first;  // the chunk's first pair
  s.turned = turned < 0 ? 0 : turned < P ? turned : P;
  if (!INTER && turned > 0 && !(P == 1 && r.interleaved)) {
    s.a = first;
    s.b = r.pairs + first;
  } else {
    s.a = 2 * first;
    s.b = s.a + P;
  }
  s.has_a = s.a + P <= channels;
  s.has_b = s.b + P <= channels;
  return s;
}

template <typename T, int P>
struct RawPairs {
  Run<T, P> a, b;
  __device__ __forceinline__ void load(const T* head, const Spot<P>& s, bool in) {
    if (in && s.has_a)
      a.load(head + s.a);
    else
      a.zero();
    if (in && s.has_b)
      b.load(head + s.b);
    else
      b.zero();
  }
  __device__ __forceinline__ void store(T* head, const Spot<P>& s) const {
    if (s.has_a) a.store(head + s.a);
    if (s.has_b) b.store(head + s.b);
  }
};
template <typename T, int P, bool INTER>
__device__ __forceinline__ Pairs<P> widen(const RawPairs<T, P>& raw) {
  Pairs<P> v;
  if constexpr (P == 1) {
    v.a.f = raw.a.get(0);
    v.b.f = raw.b.get(0);
  } else {
#pragma unroll
    for (int i = 0; i < P; i += 2) {
      if constexpr (INTER) {
        const Run<T, P>& run = i < P / 2 ? raw.a : raw.b;
        const int e = 2 * i - (i < P / 2 ? 0 : P);
        v.a.p[i / 2] = f32x2(run.get(e), run.get(e + 2));
        v.b.p[i / 2] = f32x2(run.get(e + 1), run.get(e + 3));
      } else {
        v.a.p[i / 2] = f32x2(raw.a.get(i), raw.a.get(i + 1));
        v.b.p[i / 2] = f32x2(raw.b.get(i), raw.b.get(i + 1));
      }
    }
  }
  return v;
}
template <typename T, int P, bool INTER>
__device__ __forceinline__ RawPairs<T, P> narrow(const Pairs<P>& v) {
  RawPairs<T, P> raw;
  if constexpr (P == 1) {
    raw.a.v = static_cast<T>(v.a.f);
    raw.b.v = static_cast<T>(v.b.f);
  } else {
#pragma unroll
    for (int i = 0; i < P; i += 2) {
      if constexpr (INTER) {
        Run<T, P>& run = i < P / 2 ? raw.a : raw.b;
        const int e = 2 * i - (i < P / 2 ? 0 : P);
        run.set_two(e, v.a.get(i), v.b.get(i));
        run.set_two(e + 2, v.a.get(i + 1), v.b.get(i + 1));
      } else {
        raw.a.set_two(i, v.a.get(i), v.a.get(i + 1));
        raw.b.set_two(i, v.b.get(i), v.b.get(i + 1));
      }
    }
  }
  return raw;
}

// a weight's values at a lane's pairs (1 without a weight, 0 where there is no channel)
template <int P, bool INTER>
__device__ __forceinline__ Pairs<P> weight_of(const float* weight, const Spot<P>& s) {
  if (weight == nullptr) return {Lanes<P>(1.f), Lanes<P>(1.f)};
  RawPairs<float, P> raw;
  raw.a.zero();
  raw.b.zero();
  if (s.has_a) raw.a.load_again(weight + s.a);
  if (s.has_b) raw.b.load_again(weight + s.b);
  return widen<float, P, INTER>(raw);
}

template <int P>
__device__ __forceinline__ Lanes<P> from_shared(const float* p) {
  Lanes<P> v;
  if constexpr (P == 1) {
    v.f = *p;
  } else {
#pragma unroll
    for (int i = 0; i < P / 4; ++i) {
      const float4 t = reinterpret_cast<const float4*>(p)[i];
      v.p[2 * i] = f32x2(t.x, t.y);
      v.p[2 * i + 1] = f32x2(t.z, t.w);
    }
  }
  return v;
}
template <int P>
__device__ __forceinline__ Lanes<P> negative(const Lanes<P>& v) {
  return v.each([](float f) { return -f; });
}
// the first `turned` pairs of y, the others of x: what is not turned never meets another channel's value
template <int P>
__device__ __forceinline__ void keep_unturned(Pairs<P>& y, const Pairs<P>& x, int turned) {
  if (turned == P) return;
  if constexpr (P == 1) {
    y = x;
  } else {
#pragma unroll
    for (int i = 0; i < P; i += 2) {
      y.a.p[i / 2] = f32x2(i < turned ? y.a.get(i) : x.a.get(i), i + 1 < turned ? y.a.get(i + 1) : x.a.get(i + 1));
      y.b.p[i / 2] = f32x2(i < turned ? y.b.get(i) : x.b.get(i), i + 1 < turned ? y.b.get(i + 1) : x.b.get(i + 1));
    }
  }
}

// the sum over a team of `team` lanes, a power of two
template <int U>
__device__ __forceinline__ void team_sums(float (&v)[U], int team) {
  for (int o = team / 2; o > 0; o >>= 1) {
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] += __shfl_xor_sync(0xFFFFFFFFu, v[u], o);
  }
}

// How a launch's warps share its work: items are a token's next `per` heads; teams of 2^shift lanes; `slots`
// pairs in a warp's table.
struct Plan {
  uint32_t items;
  Divisor chunks, tokens;
  int per, shift, slots;
};

// Forward. NORM: the norm and its weight. q's heads come before k's. NV runs a lane, a team apart.
template <typename T, int P, bool INTER, int NV, bool NORM>
__global__ void __launch_bounds__(kThreads) heads_kernel(const __grid_constant__ HeadsParams p, const __grid_constant__ Plan plan) {
  constexpr int U = P * NV >= 4 ? 2 : 4;  // heads of a team at a time
  extern __shared__ __align__(16) float tables[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x / 32;
  const uint32_t id = blockIdx.x * kWarps + warp;
  if (id >= plan.items) return;
  const uint32_t token = plan.chunks.quotient(id), chunk = id - token * plan.chunks.d;
  const uint32_t b = plan.tokens.quotient(token), t = token - b * plan.tokens.d;
  const int team = 1 << plan.shift, teams = 32 >> plan.shift, mine = lane >> plan.shift;
  float* cosines = tables + warp * 2 * plan.slots;
  float* sines = cosines + plan.slots;
  Spot<P> spot[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) spot[i] = spot_of<P, INTER>(p.rotary, (lane & (team - 1)) + i * team, p.channels);
  const int first = chunk * plan.per, last = min(first + plan.per, p.heads[0] + p.heads[1]);
  const float inverse_c = 1.0f / static_cast<float>(p.channels);

  RawPairs<T, P> raw[U][NV];
  const T* x = nullptr;
  auto load = [&](int which, int h, int end) {
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < NV; ++i) raw[u][i].load(x + (h + u * teams) * p.x[which].head, spot[i], h + u * teams < end);
  };
  bool fresh = true;  // no heads loaded yet
#pragma unroll 1
  for (int which = 0; which < 2; ++which) {
    const int skip = which == 0 ? 0 : p.heads[0];
    const int begin = max(first - skip, 0), end = min(last - skip, p.heads[which]);
    if (begin >= end) continue;
    const HeadView out = p.out[which];
    x = static_cast<const T*>(p.x[which].data) + b * p.x[which].batch + t * p.x[which].token;
    T* y = static_cast<T*>(out.data) + b * out.batch + t * out.token;
    load(which, begin + mine, end);
    if (fresh) find_turns(p.rotary, b * p.rotary.batch + t * p.rotary.token, plan.slots, cosines, sines);
    fresh = false;
    Pairs<P> c[NV], s[NV];  // cosines, and sines by the other channel's weight (a's negative)
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int at = ((lane & (team - 1)) + i * team) * P;
      const Lanes<P> cosine = from_shared<P>(cosines + at), sine = from_shared<P>(sines + at);
      if constexpr (NORM) {
        const Pairs<P> w = weight_of<P, INTER>(p.weight[which], spot[i]);
        c[i] = {cosine * w.a, cosine * w.b};
        s[i] = {negative(sine * w.b), sine * w.a};
      } else {
        c[i] = {cosine, cosine};
        s[i] = {negative(sine), sine};
      }
    }
#pragma unroll 1
    for (int h = begin; h < end; h += U * teams) {
      Pairs<P> v[U][NV];
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < NV; ++i) v[u][i] = widen<T, P, INTER>(raw[u][i]);
      if (h + U * teams < end) load(which, h + U * teams + mine, end);
      float rstd[U];
      if constexpr (NORM) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          rstd[u] = 0.f;
#pragma unroll
          for (int i = 0; i < NV; ++i) rstd[u] += v[u][i].a.dot(v[u][i].a) + v[u][i].b.dot(v[u][i].b);
        }
        team_sums(rstd, team);
#pragma unroll
        for (int u = 0; u < U; ++u) rstd[u] = rsqrtf(rstd[u] * inverse_c + p.eps);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int head = h + mine + u * teams;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          Pairs<P> n = v[u][i];
          if constexpr (NORM) n = {n.a * Lanes<P>(rstd[u]), n.b * Lanes<P>(rstd[u])};
          Pairs<P> turned = {fma(n.a, c[i].a, n.b * s[i].a), fma(n.b, c[i].b, n.a * s[i].b)};
          // a cosine of 1 leaves the weight
          keep_unturned(turned, {n.a * c[i].a, n.b * c[i].b}, spot[i].turned);
          if (head < end) narrow<T, P, INTER>(turned).store(y + head * out.head, spot[i]);
        }
      }
    }
  }
}

// Backward: g = dy turned back, w = g weight, xh = x rstd: dx = rstd (w - xh mean(w xh)); the first q_blocks
// blocks take q's heads, the others k's, each over its tokens. A block's sums of g xh go to row blockIdx.x of the
// partial sums.
template <typename T, int P, bool INTER, int NV>
__global__ void __launch_bounds__(kThreads)
    heads_bwd_kernel(const __grid_constant__ HeadsParams p, const __grid_constant__ Plan q_plan, const __grid_constant__ Plan k_plan,
                     int q_blocks, float* part) {
  constexpr int U = P * NV >= 4 ? 1 : 2;
  extern __shared__ __align__(16) float tables[];
  const int which = static_cast<int>(blockIdx.x) < q_blocks ? 0 : 1;
  const Plan& plan = which == 0 ? q_plan : k_plan;
  const uint32_t block = blockIdx.x - (which == 0 ? 0 : q_blocks), blocks = which == 0 ? q_blocks : gridDim.x - q_blocks;
  const int lane = threadIdx.x & 31, warp = threadIdx.x / 32;
  const int team = 1 << plan.shift, teams = 32 >> plan.shift, mine = lane >> plan.shift;
  float* cosines = tables + warp * 2 * plan.slots;
  float* sines = cosines + plan.slots;
  const HeadView xv = p.x[which], dyv = p.dy[which], outv = p.out[which];
  const float inverse_c = 1.0f / static_cast<float>(p.channels);
  Spot<P> spot[NV];
  Pairs<P> w[NV], dw[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    spot[i] = spot_of<P, INTER>(p.rotary, (lane & (team - 1)) + i * team, p.channels);
    w[i] = weight_of<P, INTER>(p.weight[which], spot[i]);
    dw[i] = {Lanes<P>(0.f), Lanes<P>(0.f)};
  }
  for (uint32_t id = block * kWarps + warp; id < plan.items; id += blocks * kWarps) {
    const uint32_t token = plan.chunks.quotient(id), chunk = id - token * plan.chunks.d;
    const uint32_t b = plan.tokens.quotient(token), t = token - b * plan.tokens.d;
    const int begin = chunk * plan.per, end = min(begin + plan.per, p.heads[which]);
    const T* x = static_cast<const T*>(xv.data) + b * xv.batch + t * xv.token;
    const T* dy = static_cast<const T*>(dyv.data) + b * dyv.batch + t * dyv.token;
    T* dx = static_cast<T*>(outv.data) + b * outv.batch + t * outv.token;
    RawPairs<T, P> raw_x[U][NV], raw_g[U][NV];
    auto load = [&](int h) {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int head = h + u * teams;
          raw_x[u][i].load(x + head * xv.head, spot[i], head < end);
          raw_g[u][i].load(dy + head * dyv.head, spot[i], head < end);
        }
    };
    load(begin + mine);
    find_turns(p.rotary, b * p.rotary.batch + t * p.rotary.token, plan.slots, cosines, sines);
    Lanes<P> c[NV], s[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int at = ((lane & (team - 1)) + i * team) * P;
      c[i] = from_shared<P>(cosines + at);
      s[i] = from_shared<P>(sines + at);
    }
#pragma unroll 1
    for (int h = begin; h < end; h += U * teams) {
      Pairs<P> v[U][NV], g[U][NV];
      float sums[2 * U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        sums[2 * u] = sums[2 * u + 1] = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          v[u][i] = widen<T, P, INTER>(raw_x[u][i]);
          const Pairs<P> d = widen<T, P, INTER>(raw_g[u][i]);
          g[u][i] = {fma(d.a, c[i], d.b * s[i]), fma(d.b, c[i], negative(d.a * s[i]))};
          keep_unturned(g[u][i], d, spot[i].turned);
          sums[2 * u] += v[u][i].a.dot(v[u][i].a) + v[u][i].b.dot(v[u][i].b);
          sums[2 * u + 1] += (v[u][i].a * w[i].a).dot(g[u][i].a) + (v[u][i].b * w[i].b).dot(g[u][i].b);
        }
      }
      if (h + U * teams < end) load(h + U * teams + mine);
      team_sums(sums, team);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int head = h + mine + u * teams;
        const float rstd = rsqrtf(sums[2 * u] * inverse_c + p.eps);
        const float along = -rstd * (sums[2 * u + 1] * rstd * inverse_c);  // -rstd mean(w xh)
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const Pairs<P> xh = {v[u][i].a * Lanes<P>(rstd), v[u][i].b * Lanes<P>(rstd)};
          if (head < end) {
            dw[i] = {fma(g[u][i].a, xh.a, dw[i].a), fma(g[u][i].b, xh.b, dw[i].b)};
            const Pairs<P> y = {fma(xh.a, Lanes<P>(along), g[u][i].a * w[i].a * Lanes<P>(rstd)),
                                fma(xh.b, Lanes<P>(along), g[u][i].b * w[i].b * Lanes<P>(rstd))};
            narrow<T, P, INTER>(y).store(dx + head * outv.head, spot[i]);
          }
        }
      }
    }
  }
  if (part == nullptr) return;
  let_next_kernel_start();
  // the warp's teams by shuffles, then the warps through shared memory, each sum in a fixed order
  __syncthreads();
  float* row = tables + warp * p.channels;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    for (int o = 16; o >= team; o >>= 1) {
      dw[i].a = dw[i].a.each([&](float f) { return f + __shfl_xor_sync(0xFFFFFFFFu, f, o); });
      dw[i].b = dw[i].b.each([&](float f) { return f + __shfl_xor_sync(0xFFFFFFFFu, f, o); });
    }
    if (mine == 0) {
#pragma unroll
      for (int j = 0; j < P; ++j) {
        if (spot[i].has_a) row[INTER && P > 1 ? spot[i].a + 2 * j : spot[i].a + j] = dw[i].a.get(j);
        if (spot[i].has_b) row[INTER && P > 1 ? spot[i].a + 2 * j + 1 : spot[i].b + j] = dw[i].b.get(j);
      }
    }
  }
  __syncthreads();
  for (int c = threadIdx.x; c < p.channels; c += kThreads) {
    float a = 0.f;
#pragma unroll
    for (int k = 0; k < kWarps; ++k) a += tables[k * p.channels + c];
    part[static_cast<int64_t>(blockIdx.x) * p.channels + c] = a;
  }
}

// a weight's gradient from the blocks' partial sums (q's rows first), in a fixed order: 32 channels a block
__global__ void __launch_bounds__(1024)
    heads_reduce_kernel(const float* __restrict__ part, float* dq_weight, float* dk_weight, int q_blocks, int blocks, int channels) {
  __shared__ float s[32][33];
  const int lane = threadIdx.x & 31, r = threadIdx.x / 32, c = blockIdx.x * 32 + lane;
  float* out = blockIdx.y == 0 ? dq_weight : dk_weight;
  const int first = blockIdx.y == 0 ? 0 : q_blocks, last = blockIdx.y == 0 ? q_blocks : blocks;
  wait_for_kernel_before();
  if (out == nullptr) return;
  float v = 0.f;
  if (c < channels)
    for (int i = first + r; i < last; i += 32) v += part[static_cast<int64_t>(i) * channels + c];
  s[r][lane] = v;
  __syncthreads();
  if (r == 0 && c < channels) {
    float a = 0.f;
#pragma unroll
    for (int k = 0; k < 32; ++k) a += s[k][lane];
    out[c] = a;
  }
}

// ------------------------------------------------------------------ launches
bool on(const HeadView& v, int elements, int size, const HeadsParams& p, int heads) {
  return (reinterpret_cast<uintptr_t>(v.data) % static_cast<uintptr_t>(elements * size < 16 ? elements * size : 16)) == 0 &&
         (p.batch <= 1 || v.batch % elements == 0) && (p.tokens <= 1 || v.token % elements == 0) && (heads <= 1 || v.head % elements == 0);
}

// whether runs of P channels are whole and aligned in every tensor of the call
bool runs_of(const HeadsParams& p, int P, int size, bool backward) {
  const RotaryParams& r = p.rotary;
  if (p.channels % (2 * P) != 0 || p.channels / (2 * P) > 32) return false;
  if (!r.interleaved && r.pairs % P != 0) return false;
  for (int i = 0; i < 2; ++i) {
    if (p.heads[i] == 0) continue;
    if (!on(p.x[i], P, size, p, p.heads[i]) || !on(p.out[i], P, size, p, p.heads[i])) return false;
    if (backward && !on(p.dy[i], P, size, p, p.heads[i])) return false;
  }
  return true;
}

// Calls f(P, INTER, NV as integral constants, lanes a team at least): runs of 16 bytes where they are whole and aligned
// (fp32 heads of more than 256 channels in two of them), else of half that, else single channels.
template <typename T, typename F>
int dispatch_heads(const HeadsParams& p, bool backward, F&& f) {
  const int size = sizeof(T);
  const auto runs = [&](auto P) {
    const int lanes = p.channels / (2 * decltype(P)::value);
    return p.rotary.interleaved ? f(P, std::true_type{}, std::integral_constant<int, 1>{}, lanes)
                                : f(P, std::false_type{}, std::integral_constant<int, 1>{}, lanes);
  };
  if (sizeof(T) == 4 && runs_of(p, 4, size, backward)) return runs(std::integral_constant<int, 4>{});
  if (runs_of(p, 8, size, backward)) return runs(std::integral_constant<int, 8>{});
  if (sizeof(T) == 2 && runs_of(p, 4, size, backward)) return runs(std::integral_constant<int, 4>{});
  const int pairs = (p.channels + 1) / 2;
  const std::integral_constant<int, 1> one;
  const std::false_type apart;
  if (pairs <= 32) return f(one, apart, std::integral_constant<int, 1>{}, pairs);
  if (pairs <= 64) return f(one, apart, std::integral_constant<int, 2>{}, 32);
  if (pairs <= 128) return f(one, apart, std::integral_constant<int, 4>{}, 32);
  return f(one, apart, std::integral_constant<int, 8>{}, 32);
}

// Items of `per` heads: all of a token's where the tokens keep the GPU's warps busy, else no more than a team
// takes at once.
Plan plan_of(const HeadsParams& p, int heads, int lanes, int run, int nv) {
  Plan plan{0, Divisor(1), Divisor(static_cast<uint32_t>(p.tokens)), heads, 0, 0};
  while ((1 << plan.shift) < lanes) ++plan.shift;
  plan.slots = (run * nv) << plan.shift;
  const int64_t tokens = static_cast<int64_t>(p.batch) * p.tokens;
  const int at_once = 32 >> plan.shift;
  int64_t chunks = (148 * 16 + tokens - 1) / tokens;
  const int64_t most = (heads + at_once - 1) / at_once;
  if (chunks > most) chunks = most;
  plan.per = static_cast<int>((heads + chunks * at_once - 1) / (chunks * at_once)) * at_once;
  chunks = (heads + plan.per - 1) / plan.per;
  plan.chunks = Divisor(static_cast<uint32_t>(chunks));
  plan.items = static_cast<uint32_t>(tokens * chunks);
  return plan;
}

template <typename T>
int heads(const HeadsParams& p, cudaStream_t stream) {
  return dispatch_heads<T>(p, false, [&](auto run, auto inter, auto nv, int lanes) {
    constexpr int P = decltype(run)::value, NV = decltype(nv)::value;
    const Plan plan = plan_of(p, p.heads[0] + p.heads[1], lanes, P, NV);
    const unsigned grid = (plan.items + kWarps - 1) / kWarps;
    const size_t smem = sizeof(float) * kWarps * 2 * plan.slots;
    auto kernel = p.norm ? heads_kernel<T, P, decltype(inter)::value, NV, true> : heads_kernel<T, P, decltype(inter)::value, NV, false>;
    kernel<<<grid, kThreads, smem, stream>>>(p, plan);
    return static_cast<int>(cudaGetLastError());
  });
}

constexpr int kMostBlocks = 148 * 2;

template <typename T>
int heads_bwd(const HeadsParams& p, float* part, cudaStream_t stream) {
  const bool sums = p.dweight[0] != nullptr || p.dweight[1] != nullptr;
  return dispatch_heads<T>(p, true, [&](auto run, auto inter, auto nv, int lanes) {
    constexpr int P = decltype(run)::value, NV = decltype(nv)::value;
    Plan plan[2] = {plan_of(p, p.heads[0] > 0 ? p.heads[0] : 1, lanes, P, NV), plan_of(p, p.heads[1] > 0 ? p.heads[1] : 1, lanes, P, NV)};
    int blocks[2];
    for (int i = 0; i < 2; ++i) {
      if (p.heads[i] == 0) plan[i].items = 0;
      const int64_t want = (static_cast<int64_t>(plan[i].items) + kWarps - 1) / kWarps;
      const int64_t share = kMostBlocks * static_cast<int64_t>(p.heads[i]) / (p.heads[0] + p.heads[1]);
      const int64_t most = share > 0 ? share : 1;
      blocks[i] = static_cast<int>(want < most ? want : most);
      if (p.dweight[i] != nullptr && blocks[i] == 0) blocks[i] = 1;  // writes zeros
    }
    size_t smem = sizeof(float) * kWarps * 2 * plan[0].slots;
    if (smem < sizeof(float) * kWarps * p.channels) smem = sizeof(float) * kWarps * p.channels;
    const int grid = blocks[0] + blocks[1];
    heads_bwd_kernel<T, P, decltype(inter)::value, NV><<<grid, kThreads, smem, stream>>>(p, plan[0], plan[1], blocks[0], sums ? part : nullptr);
    const int rc = static_cast<int>(cudaGetLastError());
    if (rc != 0 || !sums) return rc;
    return launch_after(heads_reduce_kernel, dim3((p.channels + 31) / 32, 2), 1024, 0, stream, static_cast<const float*>(part),
                        p.dweight[0], p.dweight[1], blocks[0], grid, p.channels);
  });
}

}  // namespace

size_t heads_bwd_workspace_bytes(int64_t, int, int, int channels, int) {
  return static_cast<size_t>(kMostBlocks + 2) * channels * sizeof(float);
}
int launch_heads(const HeadsParams& p, int is_f32, cudaStream_t stream) {
  return is_f32 ? heads<float>(p, stream) : heads<__nv_bfloat16>(p, stream);
}
int launch_heads_bwd(const HeadsParams& p, void* workspace, int is_f32, cudaStream_t stream) {
  float* part = static_cast<float*>(workspace);
  return is_f32 ? heads_bwd<float>(p, part, stream) : heads_bwd<__nv_bfloat16>(p, part, stream);
}

}  // namespace ffb
