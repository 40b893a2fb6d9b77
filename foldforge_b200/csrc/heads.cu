// Queries and keys of each head before an attention: divided by their root mean square, scaled by a weight,
// turned in pairs by their positions' angles, and the backward pass; the rotation alone as well.
//
// A warp takes one token's heads one after the other. A lane holds the same pairs of channels of every
// head, so it finds their angles once a token, and in the backward pass adds up the weights' gradients of
// its channels over all its tokens.
//
// Angles: a position times the pair's frequency in quarter turns in 64 bits, less the nearest whole
// number of them (exact), then sine and cosine in 32 bits of at most an eighth of a turn: a position of 2^20
// keeps the digits that a 32-bit product would lose.
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

// A pair's two channels: the turned ones first, then the others two by two (the last may stand alone).
struct Pair {
  int a, b;
};
__device__ __forceinline__ Pair pair_of(const RotaryParams& r, int j) {
  if (j < r.pairs && !r.interleaved) return {j, r.pairs + j};
  return {2 * j, 2 * j + 1};
}

template <typename T>
__device__ __forceinline__ float2 load_pair(const T* x, Pair p, int channels) {
  return make_float2(p.a < channels ? static_cast<float>(x[p.a]) : 0.f, p.b < channels ? static_cast<float>(x[p.b]) : 0.f);
}
template <typename T>
__device__ __forceinline__ void store_pair(T* x, Pair p, int channels, float2 v) {
  if (p.a < channels) x[p.a] = static_cast<T>(v.x);
  if (p.b < channels) x[p.b] = static_cast<T>(v.y);
}
__device__ __forceinline__ float2 turned(float2 v, float2 t) {
  return make_float2(v.x * t.x - v.y * t.y, v.y * t.x + v.x * t.y);
}
__device__ __forceinline__ float2 turned_back(float2 v, float2 t) { return turned(v, make_float2(t.x, -t.y)); }

struct Token {
  int64_t x, dy, out;  // element offsets of head 0
  int64_t position;
};
__device__ __forceinline__ Token token_of(const HeadsParams& p, const HeadView& x, const HeadView& dy, const HeadView& out,
                                          Divisor tokens, uint32_t id) {
  const uint32_t b = tokens.quotient(id), t = id - b * tokens.d;
  return {b * x.batch + t * x.token, b * dy.batch + t * dy.token, b * out.batch + t * out.token,
          b * p.rotary.batch + t * p.rotary.token};
}

// blockIdx.y: q or k. M pairs a lane, 32 apart.
template <typename T, int M>
__global__ void __launch_bounds__(kThreads) heads_kernel(const HeadsParams p, Divisor tokens, uint32_t total) {
  const int which = blockIdx.y, lane = threadIdx.x & 31;
  const HeadView x = p.x[which], out = p.out[which];
  const float* weight = p.weight[which];
  const float inverse_c = 1.0f / static_cast<float>(p.channels);
  for (uint32_t id = blockIdx.x * kWarps + threadIdx.x / 32; id < total; id += gridDim.x * kWarps) {
    const Token at = token_of(p, x, x, out, tokens, id);
    float2 turn[M], w[M];
#pragma unroll
    for (int m = 0; m < M; ++m) {
      const int j = lane + 32 * m;
      turn[m] = j < p.rotary.pairs ? turn_of(p.rotary, at.position, j) : make_float2(1.f, 0.f);
      w[m] = weight != nullptr ? load_pair(weight, pair_of(p.rotary, j), p.channels) : make_float2(1.f, 1.f);
    }
    for (int h = 0; h < p.heads[which]; ++h) {
      const T* in = static_cast<const T*>(x.data) + at.x + h * x.head;
      T* to = static_cast<T*>(out.data) + at.out + h * out.head;
      float2 v[M];
      float sum = 0.f;
#pragma unroll
      for (int m = 0; m < M; ++m) {
        v[m] = load_pair(in, pair_of(p.rotary, lane + 32 * m), p.channels);
        sum += v[m].x * v[m].x + v[m].y * v[m].y;
      }
      const float rstd = p.norm ? rsqrtf(warp_sum(sum) * inverse_c + p.eps) : 1.f;
      __syncwarp();
#pragma unroll
      for (int m = 0; m < M; ++m) {
        const float2 n = p.norm ? make_float2(v[m].x * rstd * w[m].x, v[m].y * rstd * w[m].y) : v[m];
        // channels behind the pairs stay what they are, also where they are not finite
        store_pair(to, pair_of(p.rotary, lane + 32 * m), p.channels,
                   lane + 32 * m < p.rotary.pairs ? turned(n, turn[m]) : n);
      }
    }
  }
}

// g = dy turned back, w = g weight, xh = x rstd: dx = rstd (w - xh mean(w xh)); a block's sums of g xh over its
// tokens and heads to row blockIdx.x of its tensor's partial sums.
template <typename T, int M>
__global__ void __launch_bounds__(kThreads)
    heads_bwd_kernel(const HeadsParams p, Divisor tokens, uint32_t total, float* part) {
  __shared__ float sums[kWarps][2 * 32 * M];
  const int which = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x / 32;
  const HeadView x = p.x[which], dy = p.dy[which], out = p.out[which];
  const float* weight = p.weight[which];
  const float inverse_c = 1.0f / static_cast<float>(p.channels);
  float2 dw[M], w[M];
#pragma unroll
  for (int m = 0; m < M; ++m) {
    dw[m] = make_float2(0.f, 0.f);
    w[m] = weight != nullptr ? load_pair(weight, pair_of(p.rotary, lane + 32 * m), p.channels) : make_float2(1.f, 1.f);
  }
  for (uint32_t id = blockIdx.x * kWarps + warp; id < total; id += gridDim.x * kWarps) {
    const Token at = token_of(p, x, dy, out, tokens, id);
    float2 turn[M];
#pragma unroll
    for (int m = 0; m < M; ++m)
      turn[m] = lane + 32 * m < p.rotary.pairs ? turn_of(p.rotary, at.position, lane + 32 * m) : make_float2(1.f, 0.f);
    for (int h = 0; h < p.heads[which]; ++h) {
      const T* in = static_cast<const T*>(x.data) + at.x + h * x.head;
      const T* gradient = static_cast<const T*>(dy.data) + at.dy + h * dy.head;
      T* to = static_cast<T*>(out.data) + at.out + h * out.head;
      float2 v[M], g[M];
      float squares = 0.f, along = 0.f;
#pragma unroll
      for (int m = 0; m < M; ++m) {
        const Pair pair = pair_of(p.rotary, lane + 32 * m);
        v[m] = load_pair(in, pair, p.channels);
        g[m] = load_pair(gradient, pair, p.channels);
        if (lane + 32 * m < p.rotary.pairs) g[m] = turned_back(g[m], turn[m]);
        squares += v[m].x * v[m].x + v[m].y * v[m].y;
        along += v[m].x * g[m].x * w[m].x + v[m].y * g[m].y * w[m].y;
      }
      const float rstd = rsqrtf(warp_sum(squares) * inverse_c + p.eps);
      const float mean = warp_sum(along) * rstd * inverse_c;  // of w xh
      __syncwarp();
#pragma unroll
      for (int m = 0; m < M; ++m) {
        const float2 xh = make_float2(v[m].x * rstd, v[m].y * rstd);
        dw[m].x += g[m].x * xh.x;
        dw[m].y += g[m].y * xh.y;
        store_pair(to, pair_of(p.rotary, lane + 32 * m), p.channels,
                   make_float2(rstd * (g[m].x * w[m].x - xh.x * mean), rstd * (g[m].y * w[m].y - xh.y * mean)));
      }
    }
  }
  if (part == nullptr) return;
  let_next_kernel_start();
#pragma unroll
  for (int m = 0; m < M; ++m) {
    const Pair pair = pair_of(p.rotary, lane + 32 * m);
    if (pair.a < p.channels) sums[warp][pair.a] = dw[m].x;
    if (pair.b < p.channels) sums[warp][pair.b] = dw[m].y;
  }
  __syncthreads();
  float* row = part + (static_cast<int64_t>(which) * gridDim.x + blockIdx.x) * p.channels;
  for (int c = threadIdx.x; c < p.channels; c += kThreads) {
    float a = 0.f;
#pragma unroll
    for (int k = 0; k < kWarps; ++k) a += sums[k][c];
    row[c] = a;
  }
}

// a weight's gradient from the blocks' partial sums, in a fixed order: 32 channels a block
__global__ void __launch_bounds__(1024)
    heads_reduce_kernel(const float* __restrict__ part, float* dq_weight, float* dk_weight, int parts, int channels) {
  __shared__ float s[32][33];
  const int lane = threadIdx.x & 31, r = threadIdx.x / 32, c = blockIdx.x * 32 + lane;
  float* out = blockIdx.y == 0 ? dq_weight : dk_weight;
  wait_for_kernel_before();
  if (out == nullptr) return;
  const float* p = part + static_cast<int64_t>(blockIdx.y) * parts * channels;
  float v = 0.f;
  if (c < channels)
    for (int i = r; i < parts; i += 32) v += p[static_cast<int64_t>(i) * channels + c];
  s[r][lane] = v;
  __syncthreads();
  if (r == 0 && c < channels) {
    float a = 0.f;
#pragma unroll
    for (int k = 0; k < 32; ++k) a += s[k][lane];
    out[c] = a;
  }
}

constexpr int kMostBlocks = 148 * 4;

int blocks_of(int64_t tokens) {
  const int64_t want = (tokens + kWarps - 1) / kWarps;
  return static_cast<int>(want < kMostBlocks ? want : kMostBlocks);
}

// Calls f(M as an integral constant), M pairs a lane for `channels`
template <typename F>
int dispatch_pairs(int channels, F&& f) {
  if (channels <= 64) return f(std::integral_constant<int, 1>{});
  if (channels <= 128) return f(std::integral_constant<int, 2>{});
  if (channels <= 256) return f(std::integral_constant<int, 4>{});
  return f(std::integral_constant<int, 8>{});
}

template <typename T>
int heads(const HeadsParams& p, cudaStream_t stream) {
  const uint32_t total = static_cast<uint32_t>(static_cast<int64_t>(p.batch) * p.tokens);
  return dispatch_pairs(p.channels, [&](auto m) {
    const dim3 grid(blocks_of(total), p.x[1].data != nullptr ? 2 : 1);
    heads_kernel<T, decltype(m)::value><<<grid, kThreads, 0, stream>>>(p, Divisor(p.tokens), total);
    return static_cast<int>(cudaGetLastError());
  });
}

template <typename T>
int heads_bwd(const HeadsParams& p, float* part, cudaStream_t stream) {
  const uint32_t total = static_cast<uint32_t>(static_cast<int64_t>(p.batch) * p.tokens);
  const bool sums = p.dweight[0] != nullptr || p.dweight[1] != nullptr;
  const dim3 grid(blocks_of(total), p.x[1].data != nullptr ? 2 : 1);
  const int rc = dispatch_pairs(p.channels, [&](auto m) {
    heads_bwd_kernel<T, decltype(m)::value><<<grid, kThreads, 0, stream>>>(p, Divisor(p.tokens), total, sums ? part : nullptr);
    return static_cast<int>(cudaGetLastError());
  });
  if (rc != 0 || !sums) return rc;
  return launch_after(heads_reduce_kernel, dim3((p.channels + 31) / 32, grid.y), 1024, 0, stream,
                      static_cast<const float*>(part), p.dweight[0], p.dweight[1], static_cast<int>(grid.x), p.channels);
}

}  // namespace

size_t heads_bwd_workspace_bytes(int64_t tokens, int, int k_heads, int channels, int) {
  return static_cast<size_t>(blocks_of(tokens)) * (k_heads > 0 ? 2 : 1) * channels * sizeof(float);
}
int launch_heads(const HeadsParams& p, int is_f32, cudaStream_t stream) {
  return is_f32 ? heads<float>(p, stream) : heads<__nv_bfloat16>(p, stream);
}
int launch_heads_bwd(const HeadsParams& p, void* workspace, int is_f32, cudaStream_t stream) {
  float* part = static_cast<float*>(workspace);
  return is_f32 ? heads_bwd<float>(p, part, stream) : heads_bwd<__nv_bfloat16>(p, part, stream);
}

}  // namespace ffb
