// Training operators bound by memory: LayerNorm forward and backward, the 8-bit checkpoint
// (mx8.cuh) packed and read back, and the gated unit silu(a) b forward and backward.
#include <type_traits>

#include "abi_util.h"
#include "common.cuh"
#include "kernels.h"
#include "mx8.cuh"

namespace ffb {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;

// Sums `v` over the GROUP threads that share a row (16, 32 or the whole block). The block form
// needs all threads; `scratch` holds one slot a warp and is used in turn (two buffers) so that one
// barrier a sum is enough.
template <int GROUP, int NSUM>
__device__ __forceinline__ void group_sum(float (&v)[NSUM], float* scratch, int& turn) {
#pragma unroll
  for (int k = 0; k < NSUM; ++k) {
#pragma unroll
    for (int o = (GROUP < 32 ? GROUP : 32) / 2; o > 0; o >>= 1) v[k] += __shfl_xor_sync(0xFFFFFFFFu, v[k], o);
  }
  if constexpr (GROUP > 32) {
    float* s = scratch + (turn & 1) * (2 * kWarps);
    turn ^= 1;
#pragma unroll
    for (int k = 0; k < NSUM; ++k)
      if ((threadIdx.x & 31) == 0) s[k * kWarps + threadIdx.x / 32] = v[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < NSUM; ++k) {
      float t = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) t += s[k * kWarps + w];
      v[k] = t;
    }
  }
}

// ------------------------------------------------------------------ LayerNorm forward
// GROUP threads hold a row in registers (NV vectors of VEC channels a thread): mean and variance
// in two passes over the registers, one read and one write an element. Writes the row's mean and
// 1 / sqrt(var + eps) in fp32 for the backward pass and, with `codes`, the input's 8-bit checkpoint.
template <typename T, int VEC, int NV, int GROUP>
__global__ void __launch_bounds__(kThreads)
    ln_train_kernel(const T* __restrict__ x, T* __restrict__ y, const float* __restrict__ gamma,
                    const float* __restrict__ beta, float* __restrict__ mean_out, float* __restrict__ rstd_out,
                    uint8_t* __restrict__ codes, uint8_t* __restrict__ scales, int64_t rows, int c, float eps) {
  constexpr int kGroups = kThreads / GROUP;
  constexpr int kLanes = kMxBlock / VEC;  // lanes that share a block of 32 channels
  __shared__ float scratch[4 * kWarps];
  int turn = 0;
  const int t = threadIdx.x % GROUP;
  const int blocks = (c + kMxBlock - 1) / kMxBlock;
  const float inv_c = 1.0f / static_cast<float>(c);
  // the loop is uniform over the block: every thread takes part in the shuffles and barriers
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * kGroups; base < rows;
       base += static_cast<int64_t>(gridDim.x) * kGroups) {
    const int64_t row = base + threadIdx.x / GROUP;
    const bool live = row < rows;
    float f[NV][VEC];
    float s[1] = {0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int col = (i * GROUP + t) * VEC;
      if (live && col < c) {
        load_vec<T, VEC>(x + row * c + col, f[i]);
      } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) f[i][j] = 0.f;
      }
#pragma unroll
      for (int j = 0; j < VEC; ++j) s[0] += f[i][j];
    }
    group_sum<GROUP>(s, scratch, turn);
    const float mean = s[0] * inv_c;
    float q[1] = {0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int col = (i * GROUP + t) * VEC;
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const float d = f[i][j] - mean;
        q[0] += col < c ? d * d : 0.f;
      }
    }
    group_sum<GROUP>(q, scratch, turn);
    const float rstd = 1.0f / sqrtf(q[0] * inv_c + eps);
    if (live && t == 0) {
      mean_out[row] = mean;
      rstd_out[row] = rstd;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int col = (i * GROUP + t) * VEC;
      const bool in = live && col < c;
      if (codes != nullptr) {
        float a = 0.f;
#pragma unroll
        for (int j = 0; j < VEC; ++j) a = fmaxf(a, mx_magnitude(f[i][j]));
        a = mx_block_max<kLanes>(a);
        const uint32_t byte = mx_scale_byte(a);
        if (in) {
          *reinterpret_cast<typename MxCodes<VEC>::type*>(codes + row * c + col) =
              mx_encode<VEC>(f[i], mx_inverse_scale(byte));
          if (t % kLanes == 0) scales[row * blocks + col / kMxBlock] = static_cast<uint8_t>(byte);
        }
      }
      if (in) {
        float o[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          o[j] = (f[i][j] - mean) * rstd;
          if (gamma != nullptr) o[j] *= gamma[col + j];
          if (beta != nullptr) o[j] += beta[col + j];
        }
        store_vec<T, VEC>(y + row * c + col, o);
      }
    }
  }
}

// ------------------------------------------------------------------ LayerNorm backward
// xh = (x - mean) rstd, w = gamma dy: dx = rstd (w - mean(w) - xh mean(w xh)) (+ residual). A thread
// keeps the same channels for every row it takes, so the sums dgamma = sum dy xh and dbeta = sum dy
// stay in its registers until the end; the block's row groups are then added in a fixed order and
// each block writes one row of partial sums, which ln_grad_reduce_kernel adds in a fixed order: the
// result does not depend on timing.
template <typename T, int VEC, int NV, int GROUP, bool MX>
__global__ void __launch_bounds__(kThreads)
    ln_bwd_kernel(const T* __restrict__ dy, const T* __restrict__ x, const uint8_t* __restrict__ codes,
                  const uint8_t* __restrict__ scales, const float* __restrict__ mean_in,
                  const float* __restrict__ rstd_in, const float* __restrict__ gamma, const T* __restrict__ residual,
                  T* __restrict__ dx, float* __restrict__ dgamma, float* __restrict__ dbeta, int64_t partial_stride,
                  int64_t rows, int c) {
  constexpr int kGroups = kThreads / GROUP;
  __shared__ float scratch[4 * kWarps];
  int turn = 0;
  const int t = threadIdx.x % GROUP;
  const int blocks = (c + kMxBlock - 1) / kMxBlock;
  const float inv_c = 1.0f / static_cast<float>(c);
  float g[NV][VEC], dg[NV][VEC], db[NV][VEC];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int col = (i * GROUP + t) * VEC;
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      g[i][j] = col >= c ? 0.f : gamma == nullptr ? 1.f : gamma[col + j];
      dg[i][j] = db[i][j] = 0.f;
    }
  }
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * kGroups; base < rows;
       base += static_cast<int64_t>(gridDim.x) * kGroups) {
    const int64_t row = base + threadIdx.x / GROUP;
    const bool live = row < rows;
    float xh[NV][VEC], w[NV][VEC];
    const float mean = live ? mean_in[row] : 0.f, rstd = live ? rstd_in[row] : 0.f;
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int col = (i * GROUP + t) * VEC;
      if (live && col < c) {
        const int64_t at = row * c + col;
        load_vec<T, VEC>(dy + at, w[i]);
        if constexpr (MX)
          mx_decode<VEC>(*reinterpret_cast<const typename MxCodes<VEC>::type*>(codes + at),
                         mx_scale(scales[row * blocks + col / kMxBlock]), xh[i]);
        else
          load_vec<T, VEC>(x + at, xh[i]);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          xh[i][j] = (xh[i][j] - mean) * rstd;
          dg[i][j] += w[i][j] * xh[i][j];
          db[i][j] += w[i][j];
          w[i][j] *= g[i][j];
          s[0] += w[i][j];
          s[1] += w[i][j] * xh[i][j];
        }
      }
    }
    group_sum<GROUP>(s, scratch, turn);
    const float c1 = s[0] * inv_c, c2 = s[1] * inv_c;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int col = (i * GROUP + t) * VEC;
      if (live && col < c) {
        const int64_t at = row * c + col;
        float o[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) o[j] = rstd * (w[i][j] - c1 - xh[i][j] * c2);
        if (residual != nullptr) {
          float r[VEC];
          load_vec<T, VEC>(residual + at, r);
#pragma unroll
          for (int j = 0; j < VEC; ++j) o[j] += r[j];
        }
        store_vec<T, VEC>(dx + at, o);
      }
    }
  }
  if (dgamma == nullptr && dbeta == nullptr) return;
  float* pg = dgamma == nullptr ? nullptr : dgamma + blockIdx.x * partial_stride;
  float* pb = dbeta == nullptr ? nullptr : dbeta + blockIdx.x * partial_stride;
  if constexpr (GROUP == kThreads) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int col = (i * GROUP + t) * VEC;
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        if (col < c && pg != nullptr) pg[col + j] = dg[i][j];
        if (col < c && pb != nullptr) pb[col + j] = db[i][j];
      }
    }
  } else {
    // the block's groups, added warp by warp into shared memory (rows of a half-warp pair first)
    __shared__ float sum[2][NV * 32 * VEC];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        if constexpr (GROUP == 16) {
          dg[i][j] += __shfl_xor_sync(0xFFFFFFFFu, dg[i][j], 16);
          db[i][j] += __shfl_xor_sync(0xFFFFFFFFu, db[i][j], 16);
        }
      }
    }
    for (int w = 0; w < kWarps; ++w) {
      if (threadIdx.x / 32 == w && (threadIdx.x & 31) < GROUP) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            const int at = (i * GROUP + t) * VEC + j;
            sum[0][at] = w == 0 ? dg[i][j] : sum[0][at] + dg[i][j];
            sum[1][at] = w == 0 ? db[i][j] : sum[1][at] + db[i][j];
          }
        }
      }
      __syncthreads();
    }
    for (int at = threadIdx.x; at < c; at += kThreads) {
      if (pg != nullptr) pg[at] = sum[0][at];
      if (pb != nullptr) pb[at] = sum[1][at];
    }
  }
}

// out[col] = sum over `parts` rows of partial sums, in a fixed order: 32 columns a block, 32 rows at
// a time, then the 32 sums of a column in turn.
__global__ void __launch_bounds__(1024)
    ln_grad_reduce_kernel(const float* __restrict__ part, float* __restrict__ dgamma, float* __restrict__ dbeta,
                          int parts, int c) {
  __shared__ float s[32][33];
  const int lane = threadIdx.x & 31, r = threadIdx.x / 32;
  const int col = blockIdx.x * 32 + lane;
  float v = 0.f;
  if (col < 2 * c)
    for (int p = r; p < parts; p += 32) v += part[static_cast<int64_t>(p) * (2 * c) + col];
  s[r][lane] = v;
  __syncthreads();
  if (r == 0 && col < 2 * c) {
    float a = 0.f;
#pragma unroll
    for (int k = 0; k < 32; ++k) a += s[k][lane];
    float* out = col < c ? dgamma : dbeta;
    if (out != nullptr) out[col < c ? col : col - c] = a;
  }
}

// ------------------------------------------------------------------ 8-bit checkpoints
// A thread takes VEC channels of a row; the lanes of a block of 32 channels agree on its largest
// magnitude by shuffles. Rows are padded to whole blocks of threads, so a block never straddles two
// rows and the lanes that share one always run together.
template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads) pack_kernel(const T* __restrict__ x, uint8_t* __restrict__ codes,
                                                         uint8_t* __restrict__ scales, int64_t rows, int c) {
  constexpr int kLanes = kMxBlock / VEC;
  const int blocks = (c + kMxBlock - 1) / kMxBlock;
  const int64_t total = rows * blocks * kLanes;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kThreads;
  for (int64_t first = static_cast<int64_t>(blockIdx.x) * kThreads; first < total; first += step) {
    const int64_t id = first + threadIdx.x;
    const int64_t block = id / kLanes;
    const int64_t row = block / blocks;
    const int col = static_cast<int>(block - row * blocks) * kMxBlock + static_cast<int>(id % kLanes) * VEC;
    const bool in = id < total && col < c;
    float f[VEC];
    float a = 0.f;
    if (in) {
      load_vec<T, VEC>(x + row * c + col, f);
#pragma unroll
      for (int j = 0; j < VEC; ++j) a = fmaxf(a, mx_magnitude(f[j]));
    }
    a = mx_block_max<kLanes>(a);
    const uint32_t byte = mx_scale_byte(a);
    if (in) {
      *reinterpret_cast<typename MxCodes<VEC>::type*>(codes + row * c + col) =
          mx_encode<VEC>(f, mx_inverse_scale(byte));
      if (id % kLanes == 0) scales[block] = static_cast<uint8_t>(byte);
    }
  }
}

template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads)
    unpack_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, T* __restrict__ x, int64_t rows,
                  int c) {
  constexpr int kLanes = kMxBlock / VEC;
  const int blocks = (c + kMxBlock - 1) / kMxBlock;
  const int64_t total = rows * blocks * kLanes;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kThreads;
  for (int64_t id = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; id < total; id += step) {
    const int64_t block = id / kLanes;
    const int64_t row = block / blocks;
    const int col = static_cast<int>(block - row * blocks) * kMxBlock + static_cast<int>(id % kLanes) * VEC;
    if (col >= c) continue;
    float f[VEC];
    mx_decode<VEC>(*reinterpret_cast<const typename MxCodes<VEC>::type*>(codes + row * c + col), mx_scale(scales[block]),
                   f);
    store_vec<T, VEC>(x + row * c + col, f);
  }
}

// ------------------------------------------------------------------ gated unit
// silu(a) and its derivative without overflow or cancellation: with t = exp(-|a| / 2) and
// r = 1 / (1 + t^2), sigmoid(|a|) = r and sigmoid(-|a|) = t^2 r. The exponential is halved because t^2
// leaves fp32's normal range at |a| = 87, where a sigmoid(a) b need not: the factors t are multiplied
// in one at a time.
struct Gate {
  float f, u, c;  // sigmoid(a) = f u, 1 - sigmoid(a) = c
  __device__ __forceinline__ explicit Gate(float a) {
    const float t = expf(-0.5f * fabsf(a));
    const float r = 1.0f / (1.0f + t * t);
    f = a >= 0.f ? 1.0f : t;
    u = f * r;
    c = a >= 0.f ? t * t * r : r;
  }
};

// h = silu(a) b for ab [rows, 2 h] = [a | b]; with `codes` (h a multiple of 32 then) also ab's 8-bit
// checkpoint.
template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads)
    swiglu_kernel(const T* __restrict__ ab, T* __restrict__ out, uint8_t* __restrict__ codes,
                  uint8_t* __restrict__ scales, int64_t rows, int h) {
  constexpr int kLanes = kMxBlock / VEC;
  const int per_row = h / VEC;
  const int64_t total = rows * per_row;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kThreads;
  for (int64_t first = static_cast<int64_t>(blockIdx.x) * kThreads; first < total; first += step) {
    const int64_t id = first + threadIdx.x;
    const bool in = id < total;
    const int64_t row = in ? id / per_row : 0;
    const int col = in ? static_cast<int>(id - row * per_row) * VEC : 0;
    float a[VEC], b[VEC];
    if (in) {
      const T* p = ab + row * 2 * h + col;
      load_vec<T, VEC>(p, a);
      load_vec<T, VEC>(p + h, b);
      float o[VEC];
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const Gate g(a[j]);
        o[j] = a[j] * g.f * g.u * b[j];
      }
      store_vec<T, VEC>(out + row * h + col, o);
    }
    if (codes != nullptr) {
      float ma = 0.f, mb = 0.f;
      if (in) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          ma = fmaxf(ma, mx_magnitude(a[j]));
          mb = fmaxf(mb, mx_magnitude(b[j]));
        }
      }
      const uint32_t ea = mx_scale_byte(mx_block_max<kLanes>(ma));
      const uint32_t eb = mx_scale_byte(mx_block_max<kLanes>(mb));
      if (in) {
        using Codes = typename MxCodes<VEC>::type;
        uint8_t* q = codes + row * 2 * h + col;
        *reinterpret_cast<Codes*>(q) = mx_encode<VEC>(a, mx_inverse_scale(ea));
        *reinterpret_cast<Codes*>(q + h) = mx_encode<VEC>(b, mx_inverse_scale(eb));
        if (threadIdx.x % kLanes == 0) {
          uint8_t* s = scales + row * (2 * h / kMxBlock) + col / kMxBlock;
          s[0] = static_cast<uint8_t>(ea);
          s[h / kMxBlock] = static_cast<uint8_t>(eb);
        }
      }
    }
  }
}

// s = sigmoid(a): da = dh b s (1 + a (1 - s)), db = dh a s, and (with `out`) h = a s b again.
template <typename T, int VEC, bool MX>
__global__ void __launch_bounds__(kThreads)
    swiglu_bwd_kernel(const T* __restrict__ dh, const T* __restrict__ ab, const uint8_t* __restrict__ codes,
                      const uint8_t* __restrict__ scales, T* __restrict__ dab, T* __restrict__ out, int64_t rows,
                      int h) {
  const int per_row = h / VEC;
  const int blocks = (2 * h + kMxBlock - 1) / kMxBlock;
  const int64_t total = rows * per_row;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kThreads;
  for (int64_t id = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; id < total; id += step) {
    const int64_t row = id / per_row;
    const int col = static_cast<int>(id - row * per_row) * VEC;
    const int64_t at = row * 2 * h + col;
    float a[VEC], b[VEC], d[VEC];
    load_vec<T, VEC>(dh + row * h + col, d);
    if constexpr (MX) {
      using Codes = typename MxCodes<VEC>::type;
      const uint8_t* s = scales + row * blocks;
      mx_decode<VEC>(*reinterpret_cast<const Codes*>(codes + at), mx_scale(s[col / kMxBlock]), a);
      mx_decode<VEC>(*reinterpret_cast<const Codes*>(codes + at + h), mx_scale(s[(col + h) / kMxBlock]), b);
    } else {
      load_vec<T, VEC>(ab + at, a);
      load_vec<T, VEC>(ab + at + h, b);
    }
    float o[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const Gate g(a[j]);
      const float unit = a[j] * g.f * g.u;
      o[j] = unit * b[j];
      const float da = d[j] * b[j] * g.f * (1.0f + a[j] * g.c) * g.u;
      b[j] = d[j] * unit;
      a[j] = da;
    }
    store_vec<T, VEC>(dab + at, a);
    store_vec<T, VEC>(dab + at + h, b);
    if (out != nullptr) store_vec<T, VEC>(out + row * h + col, o);
  }
}

// ------------------------------------------------------------------ launches
bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

int blocks_for(int64_t work, int cap) { return static_cast<int>(work < cap ? work : cap); }

// Calls f(VEC, NV, GROUP as integral constants) for rows of c channels: 16-byte vectors where the
// rows allow them (every pointer 16-byte aligned, c a whole number of vectors), the fewest threads
// that hold a row with at most 32 channels a thread.
template <typename T, typename F>
int dispatch_row(int c, bool vector, F&& f) {
  constexpr int kVec = 16 / sizeof(T);
#define FFB_ROW(V, N, G) \
  if (c <= (V) * (N) * (G)) return f(std::integral_constant<int, V>{}, std::integral_constant<int, N>{}, std::integral_constant<int, G>{})
  if (vector) {
    FFB_ROW(kVec, 1, 16);
    FFB_ROW(kVec, 1, 32);
    FFB_ROW(kVec, 2, 32);
    FFB_ROW(kVec, 3, 32);
    FFB_ROW(kVec, 4, 32);
    FFB_ROW(kVec, 1, kThreads);
    FFB_ROW(kVec, 2, kThreads);
    FFB_ROW(kVec, 32 / kVec, kThreads);
  } else {
    FFB_ROW(1, 2, 32);
    FFB_ROW(1, 8, 32);
    FFB_ROW(1, 8, kThreads);
    FFB_ROW(1, 32, kThreads);
  }
#undef FFB_ROW
  return static_cast<int>(cudaErrorInvalidValue);
}

int ln_rows_per_block(int c, int is_f32, bool vector) {
  int groups = 1;
  auto f = [&](auto, auto, auto g) {
    groups = kThreads / decltype(g)::value;
    return 0;
  };
  if (is_f32)
    dispatch_row<float>(c, vector, f);
  else
    dispatch_row<__nv_bfloat16>(c, vector, f);
  return groups;
}

constexpr int kLnBlocks = 148 * 4;  // blocks (rows of partial sums) of the backward pass at most

template <typename T>
int ln_train(const LayerNormTrain& p, cudaStream_t stream) {
  const bool vector = aligned(p.x) && aligned(p.y) && aligned(p.codes) && p.c % (16 / sizeof(T)) == 0;
  return dispatch_row<T>(p.c, vector, [&](auto v, auto n, auto g) {
    constexpr int V = decltype(v)::value, N = decltype(n)::value, G = decltype(g)::value;
    constexpr int groups = kThreads / G;
    const int grid = blocks_for((p.rows + groups - 1) / groups, 148 * 8);
    ln_train_kernel<T, V, N, G><<<grid, kThreads, 0, stream>>>(
        static_cast<const T*>(p.x), static_cast<T*>(p.y), p.gamma, p.beta, p.mean, p.rstd, p.codes, p.scales, p.rows,
        p.c, p.eps);
    return static_cast<int>(cudaGetLastError());
  });
}

template <typename T>
int ln_bwd(const LayerNormBwd& p, cudaStream_t stream) {
  const bool mx = p.codes != nullptr;
  const bool vector = aligned(p.dy) && aligned(p.dx) && aligned(p.residual) && aligned(mx ? static_cast<const void*>(p.codes) : p.x) &&
                      p.c % (16 / sizeof(T)) == 0;
  return dispatch_row<T>(p.c, vector, [&](auto v, auto n, auto g) {
    constexpr int V = decltype(v)::value, N = decltype(n)::value, G = decltype(g)::value;
    constexpr int groups = kThreads / G;
    const int grid = blocks_for((p.rows + groups - 1) / groups, kLnBlocks);
    const bool sums = p.dgamma != nullptr || p.dbeta != nullptr;
    // one block writes the gradients itself; several leave rows [dgamma | dbeta] of partial sums
    float* part = static_cast<float*>(p.workspace);
    float* dg = !sums ? nullptr : grid == 1 ? p.dgamma : part;
    float* db = !sums ? nullptr : grid == 1 ? p.dbeta : part + p.c;
    auto launch = [&](auto m) {
      ln_bwd_kernel<T, V, N, G, decltype(m)::value><<<grid, kThreads, 0, stream>>>(
          static_cast<const T*>(p.dy), static_cast<const T*>(p.x), p.codes, p.scales, p.mean, p.rstd, p.gamma,
          static_cast<const T*>(p.residual), static_cast<T*>(p.dx), dg, db, 2 * static_cast<int64_t>(p.c), p.rows, p.c);
    };
    if (mx)
      launch(std::true_type{});
    else
      launch(std::false_type{});
    if (sums && grid > 1)
      ln_grad_reduce_kernel<<<(2 * p.c + 31) / 32, 1024, 0, stream>>>(part, p.dgamma, p.dbeta, grid, p.c);
    return static_cast<int>(cudaGetLastError());
  });
}

// Calls f(VEC) for elementwise work on rows whose vectors must not straddle `multiple` channels.
template <typename T, typename F>
int dispatch_vec(bool vector, F&& f) {
  return vector ? f(std::integral_constant<int, 16 / sizeof(T)>{}) : f(std::integral_constant<int, 1>{});
}

template <typename T>
int pack(const void* x, uint8_t* codes, uint8_t* scales, int64_t rows, int c, cudaStream_t stream) {
  const bool vector = aligned(x) && aligned(codes) && c % (16 / sizeof(T)) == 0;
  return dispatch_vec<T>(vector, [&](auto v) {
    constexpr int V = decltype(v)::value;
    const int64_t threads = rows * ((c + kMxBlock - 1) / kMxBlock) * (kMxBlock / V);
    const int grid = blocks_for((threads + kThreads - 1) / kThreads, 148 * 16);
    pack_kernel<T, V><<<grid, kThreads, 0, stream>>>(static_cast<const T*>(x), codes, scales, rows, c);
    return static_cast<int>(cudaGetLastError());
  });
}

template <typename T>
int unpack(const uint8_t* codes, const uint8_t* scales, void* x, int64_t rows, int c, cudaStream_t stream) {
  const bool vector = aligned(x) && aligned(codes) && c % (16 / sizeof(T)) == 0;
  return dispatch_vec<T>(vector, [&](auto v) {
    constexpr int V = decltype(v)::value;
    const int64_t threads = rows * ((c + kMxBlock - 1) / kMxBlock) * (kMxBlock / V);
    const int grid = blocks_for((threads + kThreads - 1) / kThreads, 148 * 16);
    unpack_kernel<T, V><<<grid, kThreads, 0, stream>>>(codes, scales, static_cast<T*>(x), rows, c);
    return static_cast<int>(cudaGetLastError());
  });
}

template <typename T>
int swiglu(const void* ab, void* out, uint8_t* codes, uint8_t* scales, int64_t rows, int h, cudaStream_t stream) {
  // the fused checkpoint wants whole blocks in each half; other widths pack [a | b] in a pass of its own
  const bool fused = codes != nullptr && h % kMxBlock == 0;
  const bool vector = aligned(ab) && aligned(out) && aligned(codes) && h % (16 / sizeof(T)) == 0;
  const int rc = dispatch_vec<T>(vector, [&](auto v) {
    constexpr int V = decltype(v)::value;
    const int64_t threads = rows * (h / V);
    const int grid = blocks_for((threads + kThreads - 1) / kThreads, 148 * 16);
    swiglu_kernel<T, V><<<grid, kThreads, 0, stream>>>(static_cast<const T*>(ab), static_cast<T*>(out),
                                                       fused ? codes : nullptr, scales, rows, h);
    return static_cast<int>(cudaGetLastError());
  });
  if (rc != 0 || codes == nullptr || fused) return rc;
  return pack<T>(ab, codes, scales, rows, 2 * h, stream);
}

template <typename T>
int swiglu_bwd(const void* dh, const void* ab, const uint8_t* codes, const uint8_t* scales, void* dab, void* out,
               int64_t rows, int h, cudaStream_t stream) {
  // a vector of codes must lie in one block: in the b half that needs h to be a whole number of vectors
  const bool vector = aligned(dh) && aligned(dab) && aligned(out) && aligned(codes != nullptr ? codes : ab) &&
                      h % (16 / sizeof(T)) == 0;
  return dispatch_vec<T>(vector, [&](auto v) {
    constexpr int V = decltype(v)::value;
    const int64_t threads = rows * (h / V);
    const int grid = blocks_for((threads + kThreads - 1) / kThreads, 148 * 16);
    if (codes != nullptr)
      swiglu_bwd_kernel<T, V, true><<<grid, kThreads, 0, stream>>>(static_cast<const T*>(dh), nullptr, codes, scales,
                                                                   static_cast<T*>(dab), static_cast<T*>(out), rows, h);
    else
      swiglu_bwd_kernel<T, V, false><<<grid, kThreads, 0, stream>>>(static_cast<const T*>(dh),
                                                                    static_cast<const T*>(ab), nullptr, nullptr,
                                                                    static_cast<T*>(dab), static_cast<T*>(out), rows, h);
    return static_cast<int>(cudaGetLastError());
  });
}

}  // namespace

size_t ln_bwd_workspace_bytes(int64_t rows, int c, int is_f32) {
  // the fewest rows a block takes gives the most blocks; alignment is not known yet, so the larger of the two
  const int64_t a = ln_rows_per_block(c, is_f32, true), b = ln_rows_per_block(c, is_f32, false);
  const int64_t groups = a < b ? a : b;
  const int grid = blocks_for((rows + groups - 1) / groups, kLnBlocks);
  return static_cast<size_t>(grid) * 2 * c * sizeof(float);
}

int launch_ln_train(const LayerNormTrain& p, int is_f32, cudaStream_t stream) {
  return is_f32 ? ln_train<float>(p, stream) : ln_train<__nv_bfloat16>(p, stream);
}
int launch_ln_bwd(const LayerNormBwd& p, int is_f32, cudaStream_t stream) {
  return is_f32 ? ln_bwd<float>(p, stream) : ln_bwd<__nv_bfloat16>(p, stream);
}
int launch_checkpoint_pack(const void* x, uint8_t* codes, uint8_t* scales, int64_t rows, int c, int is_f32,
                           cudaStream_t stream) {
  return is_f32 ? pack<float>(x, codes, scales, rows, c, stream)
                : pack<__nv_bfloat16>(x, codes, scales, rows, c, stream);
}
int launch_checkpoint_unpack(const uint8_t* codes, const uint8_t* scales, void* x, int64_t rows, int c, int is_f32,
                             cudaStream_t stream) {
  return is_f32 ? unpack<float>(codes, scales, x, rows, c, stream)
                : unpack<__nv_bfloat16>(codes, scales, x, rows, c, stream);
}
int launch_swiglu_train(const void* ab, void* out, uint8_t* codes, uint8_t* scales, int64_t rows, int h, int is_f32,
                        cudaStream_t stream) {
  return is_f32 ? swiglu<float>(ab, out, codes, scales, rows, h, stream)
                : swiglu<__nv_bfloat16>(ab, out, codes, scales, rows, h, stream);
}
int launch_swiglu_bwd(const void* dh, const void* ab, const uint8_t* codes, const uint8_t* scales, void* dab, void* out,
                      int64_t rows, int h, int is_f32, cudaStream_t stream) {
  return is_f32 ? swiglu_bwd<float>(dh, ab, codes, scales, dab, out, rows, h, stream)
                : swiglu_bwd<__nv_bfloat16>(dh, ab, codes, scales, dab, out, rows, h, stream);
}

}  // namespace ffb
