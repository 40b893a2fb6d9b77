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
  for (int o = (GROUP < 32 ? GROUP : 32) / 2; o > 0; o >>= 1) {
#pragma unroll
    for (int k = 0; k < NSUM; ++k) v[k] += __shfl_xor_sync(0xFFFFFFFFu, v[k], o);
  }
  if constexpr (GROUP > 32) {
    float* s = scratch + (turn & 1) * (NSUM * kWarps);
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

// VEC values of a weight vector (fp32; 16-byte aligned where VEC > 1)
template <int VEC>
__device__ __forceinline__ void load_weight(const float* p, float (&f)[VEC]) {
  if constexpr (VEC == 1) {
    f[0] = __ldg(p);
  } else {
#pragma unroll
    for (int j = 0; j < VEC; j += 4) {
      const float4 v = __ldg(reinterpret_cast<const float4*>(p + j));
      f[j] = v.x;
      f[j + 1] = v.y;
      f[j + 2] = v.z;
      f[j + 3] = v.w;
    }
  }
}

// ------------------------------------------------------------------ LayerNorm forward
// GROUP threads hold U rows in registers (NV vectors of VEC channels a thread and row), so that U rows'
// loads are in flight at once; mean and variance in two passes over the registers, one read and one
// write an element. Writes each row's mean and 1 / sqrt(var + eps) in fp32 for the backward pass and,
// with `codes`, the input's 8-bit checkpoint.
template <typename T, int VEC, int NV, int GROUP, int U>
__global__ void __launch_bounds__(kThreads)
    ln_train_kernel(const T* __restrict__ x, T* __restrict__ y, const float* __restrict__ gamma,
                    const float* __restrict__ beta, float* __restrict__ mean_out, float* __restrict__ rstd_out,
                    uint8_t* __restrict__ codes, uint8_t* __restrict__ scales, int64_t rows, int c, float eps) {
  constexpr int kGroups = kThreads / GROUP;
  constexpr int kLanes = kMxBlock / VEC;  // lanes that share a block of 32 channels
  __shared__ float scratch[2 * U * kWarps];
  int turn = 0;
  const int t = threadIdx.x % GROUP;
  const int blocks = (c + kMxBlock - 1) / kMxBlock;
  const float inv_c = 1.0f / static_cast<float>(c);
  // rows row0 + u * kGroups; every thread takes part in the shuffles and barriers, row or not
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * (kGroups * U) + threadIdx.x / GROUP;
  typename Raw<T, VEC>::type v[U][NV];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t row = row0 + u * kGroups;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int col = (i * GROUP + t) * VEC;
      v[u][i] = row < rows && col < c ? load_raw<T, VEC>(x + row * c + col) : zero_raw<T, VEC>();
    }
  }
  float mean[U], rstd[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    mean[u] = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float f[VEC];
      widen<T, VEC>(v[u][i], f);
#pragma unroll
      for (int j = 0; j < VEC; ++j) mean[u] += f[j];
    }
  }
  group_sum<GROUP>(mean, scratch, turn);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    mean[u] *= inv_c;
    rstd[u] = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int col = (i * GROUP + t) * VEC;
      float f[VEC];
      widen<T, VEC>(v[u][i], f);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const float d = f[j] - mean[u];
        rstd[u] += col < c ? d * d : 0.f;
      }
    }
  }
  group_sum<GROUP>(rstd, scratch, turn);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    rstd[u] = rsqrtf(rstd[u] * inv_c + eps);
    const int64_t row = row0 + u * kGroups;
    if (t == 0 && row < rows) {
      mean_out[row] = mean[u];
      rstd_out[row] = rstd[u];
    }
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int col = (i * GROUP + t) * VEC;
    float w[VEC], b[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      w[j] = 1.f;
      b[j] = 0.f;
    }
    if (col < c && gamma != nullptr) load_weight<VEC>(gamma + col, w);
    if (col < c && beta != nullptr) load_weight<VEC>(beta + col, b);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t row = row0 + u * kGroups;
      const bool in = row < rows && col < c;
      float f[VEC];
      widen<T, VEC>(v[u][i], f);
      if (codes != nullptr) {
        uint32_t byte;
        const auto q = mx_quantise<T, VEC>(v[u][i], f, byte);
        if (in) {
          *reinterpret_cast<typename MxCodes<VEC>::type*>(codes + row * c + col) = q;
          if (t % kLanes == 0) scales[row * blocks + col / kMxBlock] = static_cast<uint8_t>(byte);
        }
      }
      if (in) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) f[j] = fmaf((f[j] - mean[u]) * rstd[u], w[j], b[j]);
        store_vec<T, VEC>(y + row * c + col, f);
      }
    }
  }
}

// ------------------------------------------------------------------ LayerNorm backward
// xh = (x - mean) rstd, w = gamma dy: dx = rstd (w - mean(w) - xh mean(w xh)) (+ residual). As above U
// rows of a group are in flight at once. A thread keeps the same channels for every row it takes, so
// the sums dgamma = sum dy xh and dbeta = sum dy stay in its registers until the end; the block's row
// groups are then added in a fixed order and each block writes one row of partial sums, which
// ln_grad_reduce_kernel adds in a fixed order: the result does not depend on timing.
template <typename T, int VEC, int NV, int GROUP, int U, bool MX>
__global__ void __launch_bounds__(kThreads)
    ln_bwd_kernel(const T* __restrict__ dy, const T* __restrict__ x, const uint8_t* __restrict__ codes,
                  const uint8_t* __restrict__ scales, const float* __restrict__ mean_in,
                  const float* __restrict__ rstd_in, const float* __restrict__ gamma, const T* __restrict__ residual,
                  T* __restrict__ dx, float* __restrict__ dgamma, float* __restrict__ dbeta, int64_t partial_stride,
                  int64_t rows, int c) {
  constexpr int kGroups = kThreads / GROUP;
  using Codes = typename MxCodes<VEC>::type;
  __shared__ float scratch[4 * U * kWarps];
  int turn = 0;
  const int t = threadIdx.x % GROUP;
  const int blocks = (c + kMxBlock - 1) / kMxBlock;
  const float inv_c = 1.0f / static_cast<float>(c);
  float dg[NV][VEC], db[NV][VEC];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < VEC; ++j) dg[i][j] = db[i][j] = 0.f;

  for (int64_t base = static_cast<int64_t>(blockIdx.x) * (kGroups * U); base < rows;
       base += static_cast<int64_t>(gridDim.x) * (kGroups * U)) {
    const int64_t row0 = base + threadIdx.x / GROUP;
    typename Raw<T, VEC>::type vd[U][NV], vx[MX ? 1 : U][NV];
    Codes vc[MX ? U : 1][NV];
    uint8_t vs[MX ? U : 1][NV];
    float mean[U], rstd[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t row = row0 + u * kGroups;
      const bool live = row < rows;
      mean[u] = live ? mean_in[row] : 0.f;
      rstd[u] = live ? rstd_in[row] : 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int col = (i * GROUP + t) * VEC;
        const bool in = live && col < c;
        const int64_t at = row * c + col;
        vd[u][i] = in ? load_raw<T, VEC>(dy + at) : zero_raw<T, VEC>();
        if constexpr (MX) {
          vc[u][i] = in ? __ldcs(reinterpret_cast<const Codes*>(codes + at)) : Codes{};
          vs[u][i] = in ? scales[row * blocks + col / kMxBlock] : 0;
        } else {
          vx[u][i] = in ? load_raw<T, VEC>(x + at) : zero_raw<T, VEC>();
        }
      }
    }
    // the normalised input of row u, vector i (channels past the row's end: 0 for dy, so no sum sees it)
    auto normalised = [&](int u, int i, float(&xh)[VEC]) {
      if constexpr (MX)
        mx_decode<VEC>(vc[u][i], mx_scale(vs[u][i]), xh);
      else
        widen<T, VEC>(vx[u][i], xh);
#pragma unroll
      for (int j = 0; j < VEC; ++j) xh[j] = (xh[j] - mean[u]) * rstd[u];
    };
    float s[2 * U];
#pragma unroll
    for (int u = 0; u < U; ++u) s[2 * u] = s[2 * u + 1] = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int col = (i * GROUP + t) * VEC;
      float g[VEC];
#pragma unroll
      for (int j = 0; j < VEC; ++j) g[j] = 1.f;
      if (col < c && gamma != nullptr) load_weight<VEC>(gamma + col, g);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (row0 + u * kGroups < rows && col < c) {
          float xh[VEC], d[VEC];
          normalised(u, i, xh);
          widen<T, VEC>(vd[u][i], d);
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            dg[i][j] = fmaf(d[j], xh[j], dg[i][j]);
            db[i][j] += d[j];
            const float w = d[j] * g[j];
            s[2 * u] += w;
            s[2 * u + 1] = fmaf(w, xh[j], s[2 * u + 1]);
          }
        }
      }
    }
    group_sum<GROUP>(s, scratch, turn);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int col = (i * GROUP + t) * VEC;
      float g[VEC];
#pragma unroll
      for (int j = 0; j < VEC; ++j) g[j] = 1.f;
      if (col < c && gamma != nullptr) load_weight<VEC>(gamma + col, g);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t row = row0 + u * kGroups;
        if (row < rows && col < c) {
          const float c1 = s[2 * u] * inv_c, c2 = s[2 * u + 1] * inv_c;
          const int64_t at = row * c + col;
          float xh[VEC], d[VEC];
          normalised(u, i, xh);
          widen<T, VEC>(vd[u][i], d);
#pragma unroll
          for (int j = 0; j < VEC; ++j) d[j] = rstd[u] * (d[j] * g[j] - c1 - xh[j] * c2);
          if (residual != nullptr) {
            float r[VEC];
            widen<T, VEC>(load_raw<T, VEC>(residual + at), r);
#pragma unroll
            for (int j = 0; j < VEC; ++j) d[j] += r[j];
          }
          store_vec<T, VEC>(dx + at, d);
        }
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
    // the block's groups, added warp by warp into shared memory (the two rows of a warp's halves first)
    __shared__ float sum[2][NV * 32 * VEC];
    if constexpr (GROUP == 16) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
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

// Division of 32-bit numbers below 2^31 by a fixed one: a multiplication and a shift (Granlund and
// Montgomery, "Division by invariant integers using multiplication", 1994).
struct Divisor {
  uint32_t d, m, shift;
  __host__ explicit Divisor(uint32_t n) : d(n), shift(0) {
    while ((uint64_t(1) << shift) < n) ++shift;
    m = static_cast<uint32_t>(((uint64_t(1) << 32) * ((uint64_t(1) << shift) - n)) / n + 1);
  }
  __device__ __forceinline__ uint32_t quotient(uint32_t n) const { return (__umulhi(m, n) + n) >> shift; }
};

// ------------------------------------------------------------------ 8-bit checkpoints
// A thread takes VEC channels of U places, a block's width apart, all loaded before the first is used;
// the lanes of a block of 32 channels agree on its largest magnitude by shuffles. Rows are padded to
// whole blocks (FLAT: they already are, and places follow one another in memory), so a block never
// straddles two rows and the lanes that share one always run together.
template <typename T, int VEC, bool FLAT>
struct Place {
  static constexpr int kLanes = kMxBlock / VEC;
  uint32_t block;  // of 32 channels, over all rows
  int64_t at;      // element offset
  bool in;
  __device__ __forceinline__ Place(uint32_t id, uint32_t total, int c, const Divisor& per_row) {
    block = id / kLanes;
    if constexpr (FLAT) {
      in = id < total;
      at = static_cast<int64_t>(id) * VEC;
    } else {
      const uint32_t row = per_row.quotient(block);
      const int col = static_cast<int>((block - row * per_row.d) * kMxBlock + id % kLanes * VEC);
      in = id < total && col < c;
      at = static_cast<int64_t>(row) * c + col;
    }
  }
};

template <typename T, int VEC, bool FLAT, int U>
__global__ void __launch_bounds__(kThreads) pack_kernel(const T* __restrict__ x, uint8_t* __restrict__ codes,
                                                         uint8_t* __restrict__ scales, uint32_t total, int c,
                                                         Divisor per_row) {
  using P = Place<T, VEC, FLAT>;
  const uint32_t first = blockIdx.x * (kThreads * U) + threadIdx.x;
  typename Raw<T, VEC>::type v[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const P p(first + u * kThreads, total, c, per_row);
    v[u] = p.in ? load_raw<T, VEC>(x + p.at) : zero_raw<T, VEC>();
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const P p(first + u * kThreads, total, c, per_row);
    float f[VEC];
    widen<T, VEC>(v[u], f);
    uint32_t byte;
    const auto q = mx_quantise<T, VEC>(v[u], f, byte);
    if (p.in) {
      *reinterpret_cast<typename MxCodes<VEC>::type*>(codes + p.at) = q;
      if (threadIdx.x % P::kLanes == 0) scales[p.block] = static_cast<uint8_t>(byte);
    }
  }
}

template <typename T, int VEC, bool FLAT, int U>
__global__ void __launch_bounds__(kThreads)
    unpack_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, T* __restrict__ x,
                  uint32_t total, int c, Divisor per_row) {
  using P = Place<T, VEC, FLAT>;
  using Codes = typename MxCodes<VEC>::type;
  const uint32_t first = blockIdx.x * (kThreads * U) + threadIdx.x;
  Codes v[U];
  uint8_t s[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const P p(first + u * kThreads, total, c, per_row);
    v[u] = p.in ? __ldcs(reinterpret_cast<const Codes*>(codes + p.at)) : Codes{};
    s[u] = p.in ? scales[p.block] : 0;
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const P p(first + u * kThreads, total, c, per_row);
    float f[VEC];
    mx_decode<VEC>(v[u], mx_scale(s[u]), f);
    if (p.in) store_vec<T, VEC>(x + p.at, f);
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
    const float r = __fdividef(1.0f, 1.0f + t * t);  // the divisor lies in [1, 2]: at most 2 units off
    f = a >= 0.f ? 1.0f : t;
    u = f * r;
    c = a >= 0.f ? t * t * r : r;
  }
};

// h = silu(a) b for ab [rows, 2 h] = [a | b]; with `codes` (h a multiple of 32 then) also ab's 8-bit
// checkpoint. U places a thread, as above.
template <typename T, int VEC, int U>
__global__ void __launch_bounds__(kThreads)
    swiglu_kernel(const T* __restrict__ ab, T* __restrict__ out, uint8_t* __restrict__ codes,
                  uint8_t* __restrict__ scales, uint32_t total, int h, Divisor per_row) {
  constexpr int kLanes = kMxBlock / VEC;
  const uint32_t first = blockIdx.x * (kThreads * U) + threadIdx.x;
  typename Raw<T, VEC>::type va[U], vb[U];
  int64_t at[U];  // of a
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t id = first + u * kThreads;
    const bool in = id < total;
    const uint32_t row = per_row.quotient(in ? id : 0);
    at[u] = static_cast<int64_t>(row) * 2 * h + ((in ? id : 0) - row * per_row.d) * VEC;
    va[u] = in ? load_raw<T, VEC>(ab + at[u]) : zero_raw<T, VEC>();
    vb[u] = in ? load_raw<T, VEC>(ab + at[u] + h) : zero_raw<T, VEC>();
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t id = first + u * kThreads;
    const bool in = id < total;
    float a[VEC], b[VEC];
    widen<T, VEC>(va[u], a);
    widen<T, VEC>(vb[u], b);
    if (codes != nullptr) {
      uint32_t ea, eb;
      const auto qa = mx_quantise<T, VEC>(va[u], a, ea);
      const auto qb = mx_quantise<T, VEC>(vb[u], b, eb);
      if (in) {
        *reinterpret_cast<typename MxCodes<VEC>::type*>(codes + at[u]) = qa;
        *reinterpret_cast<typename MxCodes<VEC>::type*>(codes + at[u] + h) = qb;
        if (threadIdx.x % kLanes == 0) {  // whole blocks: the scales of a row are 2 h / 32
          uint8_t* s = scales + at[u] / kMxBlock;
          s[0] = static_cast<uint8_t>(ea);
          s[h / kMxBlock] = static_cast<uint8_t>(eb);
        }
      }
    }
    if (in) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const Gate g(a[j]);
        a[j] = a[j] * g.f * g.u * b[j];
      }
      store_vec<T, VEC>(out + static_cast<int64_t>(id) * VEC, a);
    }
  }
}

// s = sigmoid(a): da = dh b s (1 + a (1 - s)), db = dh a s, and (with `out`) h = a s b again.
template <typename T, int VEC, bool MX, int U>
__global__ void __launch_bounds__(kThreads)
    swiglu_bwd_kernel(const T* __restrict__ dh, const T* __restrict__ ab, const uint8_t* __restrict__ codes,
                      const uint8_t* __restrict__ scales, T* __restrict__ dab, T* __restrict__ out, uint32_t total,
                      int h, Divisor per_row) {
  using Codes = typename MxCodes<VEC>::type;
  const int blocks = (2 * h + kMxBlock - 1) / kMxBlock;
  const uint32_t first = blockIdx.x * (kThreads * U) + threadIdx.x;
  typename Raw<T, VEC>::type vd[U], va[MX ? 1 : U], vb[MX ? 1 : U];
  Codes ca[MX ? U : 1], cb[MX ? U : 1];
  uint8_t sa[MX ? U : 1], sb[MX ? U : 1];
  int64_t at[U];  // of a and da
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t id = first + u * kThreads;
    const bool in = id < total;
    const uint32_t row = per_row.quotient(in ? id : 0);
    const int col = static_cast<int>(((in ? id : 0) - row * per_row.d) * VEC);
    at[u] = static_cast<int64_t>(row) * 2 * h + col;
    vd[u] = in ? load_raw<T, VEC>(dh + static_cast<int64_t>(id) * VEC) : zero_raw<T, VEC>();
    if constexpr (MX) {
      const uint8_t* s = scales + static_cast<int64_t>(row) * blocks;
      ca[u] = in ? __ldcs(reinterpret_cast<const Codes*>(codes + at[u])) : Codes{};
      cb[u] = in ? __ldcs(reinterpret_cast<const Codes*>(codes + at[u] + h)) : Codes{};
      sa[u] = in ? s[col / kMxBlock] : 0;
      sb[u] = in ? s[(col + h) / kMxBlock] : 0;
    } else {
      va[u] = in ? load_raw<T, VEC>(ab + at[u]) : zero_raw<T, VEC>();
      vb[u] = in ? load_raw<T, VEC>(ab + at[u] + h) : zero_raw<T, VEC>();
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t id = first + u * kThreads;
    if (id >= total) continue;
    float a[VEC], b[VEC], d[VEC];
    widen<T, VEC>(vd[u], d);
    if constexpr (MX) {
      mx_decode<VEC>(ca[u], mx_scale(sa[u]), a);
      mx_decode<VEC>(cb[u], mx_scale(sb[u]), b);
    } else {
      widen<T, VEC>(va[u], a);
      widen<T, VEC>(vb[u], b);
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
    store_vec<T, VEC>(dab + at[u], a);
    store_vec<T, VEC>(dab + at[u] + h, b);
    if (out != nullptr) store_vec<T, VEC>(out + static_cast<int64_t>(id) * VEC, o);
  }
}

// ------------------------------------------------------------------ launches
bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// How a row of c channels is held: 16-byte vectors where the rows allow them (every pointer 16-byte
// aligned, c a whole number of vectors), the fewest threads that hold it with at most 32 channels a
// thread, and U rows at a time where a row leaves few registers in use. Calls
// f(VEC, NV, GROUP, U as integral constants).
template <typename T, typename F>
int dispatch_row(int c, bool vector, F&& f) {
  constexpr int kVec = 16 / sizeof(T);
#define FFB_ROW(V, N, G, U)                                                                                   \
  if (c <= (V) * (N) * (G))                                                                                   \
  return f(std::integral_constant<int, V>{}, std::integral_constant<int, N>{}, std::integral_constant<int, G>{}, \
           std::integral_constant<int, U>{})
  if (vector) {
    FFB_ROW(kVec, 1, 16, 4);
    FFB_ROW(kVec, 1, 32, 4);
    FFB_ROW(kVec, 2, 32, 2);
    FFB_ROW(kVec, 3, 32, 2);
    FFB_ROW(kVec, 4, 32, 1);
    FFB_ROW(kVec, 1, kThreads, 4);
    FFB_ROW(kVec, 2, kThreads, 2);
    FFB_ROW(kVec, 32 / kVec, kThreads, 1);
  } else {
    FFB_ROW(1, 2, 32, 4);
    FFB_ROW(1, 8, 32, 2);
    FFB_ROW(1, 8, kThreads, 2);
    FFB_ROW(1, 32, kThreads, 1);
  }
#undef FFB_ROW
  return static_cast<int>(cudaErrorInvalidValue);
}

constexpr int kLnBlocks = 148 * 2;  // blocks (rows of partial sums) of the backward pass at most

template <typename T>
int ln_bwd_blocks(int64_t rows, int c, bool vector) {
  int blocks = 0;
  dispatch_row<T>(c, vector, [&](auto, auto, auto g, auto u) {
    constexpr int per = kThreads / decltype(g)::value * decltype(u)::value;  // rows a block takes at a time
    const int64_t want = (rows + per - 1) / per;
    blocks = static_cast<int>(want < kLnBlocks ? want : kLnBlocks);
    return 0;
  });
  return blocks;
}

template <typename T>
int ln_train(const LayerNormTrain& p, cudaStream_t stream) {
  const bool vector = aligned(p.x) && aligned(p.y) && aligned(p.codes) && aligned(p.gamma) && aligned(p.beta) &&
                      p.c % (16 / sizeof(T)) == 0;
  return dispatch_row<T>(p.c, vector, [&](auto v, auto n, auto g, auto u) {
    constexpr int V = decltype(v)::value, N = decltype(n)::value, G = decltype(g)::value, U = decltype(u)::value;
    constexpr int per = kThreads / G * U;
    // a launch's grid is 31 bits wide
    for (int64_t first = 0; first < p.rows; first += int64_t(1) << 30) {
      const int64_t rows = p.rows - first < (int64_t(1) << 30) ? p.rows - first : int64_t(1) << 30;
      ln_train_kernel<T, V, N, G, U><<<static_cast<int>((rows + per - 1) / per), kThreads, 0, stream>>>(
          static_cast<const T*>(p.x) + first * p.c, static_cast<T*>(p.y) + first * p.c, p.gamma, p.beta, p.mean + first,
          p.rstd + first, p.codes == nullptr ? nullptr : p.codes + first * p.c,
          p.codes == nullptr ? nullptr : p.scales + first * ((p.c + kMxBlock - 1) / kMxBlock), rows, p.c, p.eps);
    }
    return static_cast<int>(cudaGetLastError());
  });
}

template <typename T>
int ln_bwd(const LayerNormBwd& p, cudaStream_t stream) {
  const bool mx = p.codes != nullptr;
  const bool vector = aligned(p.dy) && aligned(p.dx) && aligned(p.residual) && aligned(p.gamma) &&
                      aligned(mx ? static_cast<const void*>(p.codes) : p.x) && p.c % (16 / sizeof(T)) == 0;
  const int grid = ln_bwd_blocks<T>(p.rows, p.c, vector);
  return dispatch_row<T>(p.c, vector, [&](auto v, auto n, auto g, auto u) {
    constexpr int V = decltype(v)::value, N = decltype(n)::value, G = decltype(g)::value, U = decltype(u)::value;
    const bool sums = p.dgamma != nullptr || p.dbeta != nullptr;
    // one block writes the gradients itself; several leave rows [dgamma | dbeta] of partial sums
    float* part = static_cast<float*>(p.workspace);
    float* dg = !sums ? nullptr : grid == 1 ? p.dgamma : part;
    float* db = !sums ? nullptr : grid == 1 ? p.dbeta : part + p.c;
    auto launch = [&](auto m) {
      ln_bwd_kernel<T, V, N, G, U, decltype(m)::value><<<grid, kThreads, 0, stream>>>(
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

// Elementwise work on `rows` rows of `per_row` units (vectors, or blocks of 32 channels times their
// lanes): launches f(first row, rows) on pieces whose unit numbers stay below 2^30, so that the kernels
// divide 32-bit numbers.
template <typename F>
int in_pieces(int64_t rows, int64_t per_row, F&& f) {
  const int64_t most = (int64_t(1) << 30) / per_row > 0 ? (int64_t(1) << 30) / per_row : 1;
  for (int64_t first = 0; first < rows; first += most) f(first, rows - first < most ? rows - first : most);
  return static_cast<int>(cudaGetLastError());
}

constexpr int kUnits = 4;  // units a thread takes

// Calls f(VEC, FLAT) for the checkpoint kernels: vectors where the rows allow them, and whether rows
// are whole blocks.
template <typename T, typename F>
int dispatch_checkpoint(int c, bool vector, F&& f) {
  constexpr int kVec = 16 / sizeof(T);
  if (!vector) return f(std::integral_constant<int, 1>{}, std::false_type{});
  if (c % kMxBlock == 0) return f(std::integral_constant<int, kVec>{}, std::true_type{});
  return f(std::integral_constant<int, kVec>{}, std::false_type{});
}

template <typename T>
int pack(const void* x, uint8_t* codes, uint8_t* scales, int64_t rows, int c, cudaStream_t stream) {
  const bool vector = aligned(x) && aligned(codes) && c % (16 / sizeof(T)) == 0;
  const int blocks = (c + kMxBlock - 1) / kMxBlock;
  return dispatch_checkpoint<T>(c, vector, [&](auto v, auto flat) {
    constexpr int V = decltype(v)::value;
    constexpr bool FLAT = decltype(flat)::value;
    const int64_t units = static_cast<int64_t>(blocks) * (kMxBlock / V);
    return in_pieces(rows, units, [&](int64_t first, int64_t n) {
      const uint32_t total = static_cast<uint32_t>(n * units);
      pack_kernel<T, V, FLAT, kUnits><<<(total + kThreads * kUnits - 1) / (kThreads * kUnits), kThreads, 0, stream>>>(
          static_cast<const T*>(x) + first * c, codes + first * c, scales + first * blocks, total, c, Divisor(blocks));
    });
  });
}

template <typename T>
int unpack(const uint8_t* codes, const uint8_t* scales, void* x, int64_t rows, int c, cudaStream_t stream) {
  const bool vector = aligned(x) && aligned(codes) && c % (16 / sizeof(T)) == 0;
  const int blocks = (c + kMxBlock - 1) / kMxBlock;
  return dispatch_checkpoint<T>(c, vector, [&](auto v, auto flat) {
    constexpr int V = decltype(v)::value;
    constexpr bool FLAT = decltype(flat)::value;
    const int64_t units = static_cast<int64_t>(blocks) * (kMxBlock / V);
    return in_pieces(rows, units, [&](int64_t first, int64_t n) {
      const uint32_t total = static_cast<uint32_t>(n * units);
      unpack_kernel<T, V, FLAT, kUnits><<<(total + kThreads * kUnits - 1) / (kThreads * kUnits), kThreads, 0, stream>>>(
          codes + first * c, scales + first * blocks, static_cast<T*>(x) + first * c, total, c, Divisor(blocks));
    });
  });
}

template <typename T, typename F>
int dispatch_vec(bool vector, F&& f) {
  return vector ? f(std::integral_constant<int, 16 / sizeof(T)>{}) : f(std::integral_constant<int, 1>{});
}

template <typename T>
int swiglu(const void* ab, void* out, uint8_t* codes, uint8_t* scales, int64_t rows, int h, cudaStream_t stream) {
  // the fused checkpoint wants whole blocks in each half; other widths pack [a | b] in a pass of its own
  const bool fused = codes != nullptr && h % kMxBlock == 0;
  const bool vector = aligned(ab) && aligned(out) && aligned(codes) && h % (16 / sizeof(T)) == 0;
  const int rc = dispatch_vec<T>(vector, [&](auto v) {
    constexpr int V = decltype(v)::value;
    return in_pieces(rows, h / V, [&](int64_t first, int64_t n) {
      const uint32_t total = static_cast<uint32_t>(n * (h / V));
      swiglu_kernel<T, V, 2><<<(total + kThreads * 2 - 1) / (kThreads * 2), kThreads, 0, stream>>>(
          static_cast<const T*>(ab) + first * 2 * h, static_cast<T*>(out) + first * h,
          fused ? codes + first * 2 * h : nullptr, fused ? scales + first * (2 * h / kMxBlock) : nullptr, total, h,
          Divisor(h / V));
    });
  });
  if (rc != 0 || codes == nullptr || fused) return rc;
  return pack<T>(ab, codes, scales, rows, 2 * h, stream);
}

template <typename T>
int swiglu_bwd(const void* dh, const void* ab, const uint8_t* codes, const uint8_t* scales, void* dab, void* out,
               int64_t rows, int h, cudaStream_t stream) {
  // h is a whole number of vectors: one of b's codes then lies in one block of 32 as well
  const bool vector = aligned(dh) && aligned(dab) && aligned(out) && aligned(codes != nullptr ? codes : ab) &&
                      h % (16 / sizeof(T)) == 0;
  const int blocks = (2 * h + kMxBlock - 1) / kMxBlock;
  return dispatch_vec<T>(vector, [&](auto v) {
    constexpr int V = decltype(v)::value;
    return in_pieces(rows, h / V, [&](int64_t first, int64_t n) {
      const uint32_t total = static_cast<uint32_t>(n * (h / V));
      const int grid = static_cast<int>((total + kThreads * 2 - 1) / (kThreads * 2));
      const T* g = static_cast<const T*>(dh) + first * h;
      T* d = static_cast<T*>(dab) + first * 2 * h;
      T* o = out == nullptr ? nullptr : static_cast<T*>(out) + first * h;
      if (codes != nullptr)
        swiglu_bwd_kernel<T, V, true, 2><<<grid, kThreads, 0, stream>>>(g, nullptr, codes + first * 2 * h,
                                                                        scales + first * blocks, d, o, total, h,
                                                                        Divisor(h / V));
      else
        swiglu_bwd_kernel<T, V, false, 2><<<grid, kThreads, 0, stream>>>(
            g, static_cast<const T*>(ab) + first * 2 * h, nullptr, nullptr, d, o, total, h, Divisor(h / V));
    });
  });
}

}  // namespace

size_t ln_bwd_workspace_bytes(int64_t rows, int c, int is_f32) {
  // the tensors' alignment is not known here: room for the form with more blocks
  const int a = is_f32 ? ln_bwd_blocks<float>(rows, c, true) : ln_bwd_blocks<__nv_bfloat16>(rows, c, true);
  const int b = is_f32 ? ln_bwd_blocks<float>(rows, c, false) : ln_bwd_blocks<__nv_bfloat16>(rows, c, false);
  const int blocks = a > b ? a : b;
  return blocks > 1 ? static_cast<size_t>(blocks) * 2 * c * sizeof(float) : 0;
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
