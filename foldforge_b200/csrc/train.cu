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
    for (int i = 0; i < NV; ++i) mean[u] += widen<T, VEC>(v[u][i]).sum();
  }
  group_sum<GROUP>(mean, scratch, turn);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    mean[u] *= inv_c;
    rstd[u] = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const Lanes<VEC> d = widen<T, VEC>(v[u][i]) + Lanes<VEC>(-mean[u]);
      rstd[u] += (i * GROUP + t) * VEC < c ? (d * d).sum() : 0.f;
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
    const Lanes<VEC> w = col < c && gamma != nullptr ? load_weight<VEC>(gamma + col) : Lanes<VEC>(1.f);
    const Lanes<VEC> b = col < c && beta != nullptr ? load_weight<VEC>(beta + col) : Lanes<VEC>(0.f);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t row = row0 + u * kGroups;
      const bool in = row < rows && col < c;
      const Lanes<VEC> f = widen<T, VEC>(v[u][i]);
      if (codes != nullptr) {
        uint32_t byte;
        const auto q = mx_quantise<T, VEC>(v[u][i], f, byte);
        if (in) {
          *reinterpret_cast<typename MxCodes<VEC>::type*>(codes + row * c + col) = q;
          if (t % kLanes == 0) scales[row * blocks + col / kMxBlock] = static_cast<uint8_t>(byte);
        }
      }
      if (in)
        store_lanes<T, VEC>(y + row * c + col, fma((f + Lanes<VEC>(-mean[u])) * Lanes<VEC>(rstd[u]), w, b));
    }
  }
}

// The block's sums of each channel over its rows (dg, db: a thread's, over the rows it took) to row
// blockIdx.x of the partial sums. `space` holds kWarps NV GROUP VEC floats unless the whole block shares
// each row, and nobody uses it any more once the block has come here.
template <int VEC, int NV, int GROUP>
__device__ __forceinline__ void write_column_sums(Lanes<VEC> (&dg)[NV], Lanes<VEC> (&db)[NV], float* dgamma, float* dbeta,
                                                  int64_t partial_stride, int c, float* space) {
  if (dgamma == nullptr && dbeta == nullptr) return;
  const int t = threadIdx.x % GROUP;
  float* pg = dgamma == nullptr ? nullptr : dgamma + blockIdx.x * partial_stride;
  float* pb = dbeta == nullptr ? nullptr : dbeta + blockIdx.x * partial_stride;
  if constexpr (GROUP == kThreads) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int col = (i * GROUP + t) * VEC;
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        if (col < c && pg != nullptr) pg[col + j] = dg[i].get(j);
        if (col < c && pb != nullptr) pb[col + j] = db[i].get(j);
      }
    }
  } else {
    // a warp's groups by shuffles, then the warps through shared memory, each sum in a fixed order
    constexpr int kColumns = NV * GROUP * VEC;
    const int warp = threadIdx.x / 32;
#pragma unroll
    for (int o = 16; o >= GROUP; o >>= 1) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        dg[i] = dg[i].each([&](float v) { return v + __shfl_xor_sync(0xFFFFFFFFu, v, o); });
        db[i] = db[i].each([&](float v) { return v + __shfl_xor_sync(0xFFFFFFFFu, v, o); });
      }
    }
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      __syncthreads();
      if ((threadIdx.x & 31) < GROUP) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
          for (int j = 0; j < VEC; ++j)
            space[warp * kColumns + (i * GROUP + t) * VEC + j] = which == 0 ? dg[i].get(j) : db[i].get(j);
      }
      __syncthreads();
      float* out = which == 0 ? pg : pb;
      for (int at = threadIdx.x; at < c && out != nullptr; at += kThreads) {
        float a = 0.f;
#pragma unroll
        for (int k = 0; k < kWarps; ++k) a += space[k * kColumns + at];
        out[at] = a;
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
  Lanes<VEC> dg[NV], db[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) dg[i] = db[i] = Lanes<VEC>(0.f);

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
    // The normalised input of row u, vector i. The mean is taken off first: x rstd - mean rstd would leave
    // rounding errors of mean rstd where a row hardly varies.
    auto normalised = [&](int u, int i) {
      const Lanes<VEC> centre(-mean[u]), r(rstd[u]);
      if constexpr (MX)
        return fma(mx_codes_value<VEC>(vc[u][i]), Lanes<VEC>(mx_scale(vs[u][i])), centre) * r;
      else
        return (widen<T, VEC>(vx[u][i]) + centre) * r;
    };
    float s[2 * U];
#pragma unroll
    for (int u = 0; u < U; ++u) s[2 * u] = s[2 * u + 1] = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int col = (i * GROUP + t) * VEC;
      const Lanes<VEC> g = col < c && gamma != nullptr ? load_weight<VEC>(gamma + col) : Lanes<VEC>(1.f);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (row0 + u * kGroups < rows && col < c) {
          const Lanes<VEC> xh = normalised(u, i), d = widen<T, VEC>(vd[u][i]), w = d * g;
          dg[i] = fma(d, xh, dg[i]);
          db[i] = db[i] + d;
          s[2 * u] += w.sum();
          s[2 * u + 1] += (w * xh).sum();
        }
      }
    }
    group_sum<GROUP>(s, scratch, turn);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int col = (i * GROUP + t) * VEC;
      const Lanes<VEC> g = col < c && gamma != nullptr ? load_weight<VEC>(gamma + col) : Lanes<VEC>(1.f);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t row = row0 + u * kGroups;
        if (row < rows && col < c) {
          const float c1 = s[2 * u] * inv_c, c2 = s[2 * u + 1] * inv_c;
          const int64_t at = row * c + col;
          const Lanes<VEC> w = widen<T, VEC>(vd[u][i]) * g;
          Lanes<VEC> o = fma(normalised(u, i), Lanes<VEC>(-c2), w + Lanes<VEC>(-c1)) * Lanes<VEC>(rstd[u]);
          if (residual != nullptr) o = o + widen<T, VEC>(load_raw<T, VEC>(residual + at));
          store_lanes<T, VEC>(dx + at, o);
        }
      }
    }
  }
  __shared__ float space[GROUP == kThreads ? 1 : kWarps * NV * GROUP * VEC];
  write_column_sums<VEC, NV, GROUP>(dg, db, dgamma, dbeta, partial_stride, c, space);
}

// ------------------------------------------------------------------ LayerNorm, rows streamed
// The same sums where rows are whole 16-byte words (c a multiple of 16): a team (a warp, or the block for
// rows that a warp's registers cannot hold) takes RS = rows at a time, which lie next to one another in
// memory, and has them copied to its own ring of kRing slots in shared memory by bulk copies. The loads in
// flight then do not depend on registers or occupancy, and cost one thread a few instructions.
constexpr int kRing = 3;

template <int TEAM>
__device__ __forceinline__ void team_sync() {
  if constexpr (TEAM == 32)
    __syncwarp();
  else
    __syncthreads();
}

// whether all of a team's threads say so, as all of them learn
template <int TEAM>
__device__ __forceinline__ bool team_all(bool yes) {
  if constexpr (TEAM == 32)
    return __all_sync(0xFFFFFFFFu, yes);
  else
    return __syncthreads_and(yes);
}

// A team's ring: `streams` tensors with rows of row_bytes[k] bytes; a slot holds RS rows of each, one
// tensor after the other.
template <int TEAM, int RS>
struct Ring {
  uint8_t* slots;
  uint64_t* full;
  int streams, slot_bytes;
  const uint8_t* base[3];
  int row_bytes[3];
  int64_t rows, teams, first;  // this team's chunks of RS rows: first, first + teams, ..

  __device__ __forceinline__ Ring(uint8_t* smem, uint64_t* bars, int64_t all_rows) : streams(0), slot_bytes(0), rows(all_rows) {
    constexpr int kTeams = kThreads / TEAM;
    const int team = threadIdx.x / TEAM;
    slots = smem;
    full = bars + team * kRing;
    teams = static_cast<int64_t>(gridDim.x) * kTeams;
    first = static_cast<int64_t>(blockIdx.x) * kTeams + team;
    if (threadIdx.x % TEAM == 0) {
      for (int i = 0; i < kRing; ++i) mbar_init(&full[i], 1);
      fence_mbar_init();
    }
  }
  __device__ __forceinline__ void add(const void* p, int bytes) {
    base[streams] = static_cast<const uint8_t*>(p);
    row_bytes[streams] = bytes;
    slot_bytes += RS * bytes;
    ++streams;
  }
  // after the last add: the team's part of shared memory
  __device__ __forceinline__ void place() { slots += static_cast<int64_t>(threadIdx.x / TEAM) * kRing * slot_bytes; }
  __device__ __forceinline__ int64_t row(int turn) const { return (first + turn * teams) * RS; }
  // one thread: the copies of the team's chunk number `turn`
  __device__ __forceinline__ void fetch(int turn) {
    const int64_t at = row(turn);
    if (at >= rows) return;
    const int n = rows - at < RS ? static_cast<int>(rows - at) : RS;
    uint64_t* bar = &full[turn % kRing];
    uint8_t* dst = slots + turn % kRing * slot_bytes;
    int bytes = 0;
#pragma unroll
    for (int k = 0; k < 3; ++k)
      if (k < streams) bytes += n * row_bytes[k];
    mbar_arrive_expect_tx(bar, bytes);
#pragma unroll
    for (int k = 0; k < 3; ++k)
      if (k < streams) {
        bulk_load(dst, base[k] + at * row_bytes[k], n * row_bytes[k], bar);
        dst += RS * row_bytes[k];
      }
  }
  // False (for the whole team) where the copies never came: the error word says so, and the other slots'
  // copies have had the same time to land.
  __device__ __forceinline__ bool wait(int turn, int* err) {
    return team_all<TEAM>(mbar_wait(&full[turn % kRing], (turn / kRing) & 1, err, kErrTimeoutLoad));
  }
  // row r of a slot's tensor k (whose rows follow those of the tensors before it)
  template <typename P>
  __device__ __forceinline__ const P* at(int turn, int offset) const {
    return reinterpret_cast<const P*>(slots + turn % kRing * slot_bytes + offset);
  }
};

// FULL: c fills the group's vectors, so that no lane has to look whether its channels are there.
template <typename T, int VEC, int NV, int GROUP, int U, bool FULL>
__global__ void __launch_bounds__(kThreads, NV * VEC * sizeof(T) <= 32 ? 2 : 1)
    ln_train_stream_kernel(const T* __restrict__ x, T* __restrict__ y, const float* __restrict__ gamma,
                           const float* __restrict__ beta, float* __restrict__ mean_out, float* __restrict__ rstd_out,
                           uint8_t* __restrict__ codes, uint8_t* __restrict__ scales, int64_t rows, int c, float eps,
                           int* err) {
  constexpr int kTeam = GROUP <= 32 ? 32 : kThreads;
  constexpr int kGroups = kTeam / GROUP;  // rows of a team side by side
  constexpr int RS = kGroups * U;
  constexpr int kLanes = kMxBlock / VEC;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint64_t bars[kThreads / kTeam * kRing];
  __shared__ float scratch[2 * U * kWarps];
  int turn_of = 0;
  const int t = threadIdx.x % GROUP, g = threadIdx.x % kTeam / GROUP;
  const bool leader = threadIdx.x % kTeam == 0;
  const int blocks = (c + kMxBlock - 1) / kMxBlock;
  const float inv_c = 1.0f / static_cast<float>(c);
  Ring<kTeam, RS> ring(smem, bars, rows);
  ring.add(x, c * static_cast<int>(sizeof(T)));
  ring.place();
  __syncthreads();
  if (leader)
    for (int i = 0; i < kRing; ++i) ring.fetch(i);
  Lanes<VEC> w[NV], b[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int col = (i * GROUP + t) * VEC;
    w[i] = (FULL || col < c) && gamma != nullptr ? load_weight<VEC>(gamma + col) : Lanes<VEC>(1.f);
    b[i] = (FULL || col < c) && beta != nullptr ? load_weight<VEC>(beta + col) : Lanes<VEC>(0.f);
  }
  for (int turn = 0; ring.row(turn) < rows; ++turn) {
    if (!ring.wait(turn, err)) break;
    const int64_t row0 = ring.row(turn) + g;
    const T* have = ring.template at<T>(turn, 0) + g * c;
    // a row past the last one reads what the slot held before, and nothing of it is kept
    auto read = [&](int u, int i) {
      const int col = (i * GROUP + t) * VEC;
      return FULL || col < c ? shared_raw<T, VEC>(have + u * kGroups * c + col) : zero_raw<T, VEC>();
    };
    auto squares = [&](const Lanes<VEC>& f, float m, int i) {
      const Lanes<VEC> d = f + Lanes<VEC>(-m);
      const float q = d.dot(d);
      return FULL || (i * GROUP + t) * VEC < c ? q : 0.f;
    };
    auto finish = [&](const typename Raw<T, VEC>::type& v, const Lanes<VEC>& f, float m, float r, int64_t row, int i) {
      const int col = (i * GROUP + t) * VEC;
      const bool in = row < rows && (FULL || col < c);
      if (codes != nullptr) {
        uint32_t byte;
        const auto q = mx_quantise<T, VEC>(v, f, byte);
        if (in) {
          *reinterpret_cast<typename MxCodes<VEC>::type*>(codes + row * c + col) = q;
          if (t % kLanes == 0) scales[row * blocks + col / kMxBlock] = static_cast<uint8_t>(byte);
        }
      }
      if (in) store_lanes<T, VEC>(y + row * c + col, fma((f + Lanes<VEC>(-m)) * Lanes<VEC>(r), w[i], b[i]));
    };
    auto keep = [&](float m, float r, int64_t row) {
      if (t == 0 && row < rows) {
        mean_out[row] = m;
        rstd_out[row] = r;
      }
    };
    if constexpr (GROUP > 32) {
      // the block's barriers cost more than reading the slot again: all rows of the chunk at a time
      float m[U], r[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        m[u] = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) m[u] += widen<T, VEC>(read(u, i)).sum();
      }
      group_sum<GROUP>(m, scratch, turn_of);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        m[u] *= inv_c;
        r[u] = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) r[u] += squares(widen<T, VEC>(read(u, i)), m[u], i);
      }
      group_sum<GROUP>(r, scratch, turn_of);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        r[u] = rsqrtf(r[u] * inv_c + eps);
        keep(m[u], r[u], row0 + u);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const auto v = read(u, i);
          finish(v, widen<T, VEC>(v), m[u], r[u], row0 + u, i);
        }
      }
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t row = row0 + u * kGroups;
        typename Raw<T, VEC>::type v[NV];
        Lanes<VEC> f[NV];
        float m[1] = {0.f}, r[1] = {0.f};
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          v[i] = read(u, i);
          f[i] = widen<T, VEC>(v[i]);
          m[0] += f[i].sum();
        }
        group_sum<GROUP>(m, scratch, turn_of);
        m[0] *= inv_c;
#pragma unroll
        for (int i = 0; i < NV; ++i) r[0] += squares(f[i], m[0], i);
        group_sum<GROUP>(r, scratch, turn_of);
        r[0] = rsqrtf(r[0] * inv_c + eps);
        keep(m[0], r[0], row);
#pragma unroll
        for (int i = 0; i < NV; ++i) finish(v[i], f[i], m[0], r[0], row, i);
      }
    }
    team_sync<kTeam>();
    if (leader) ring.fetch(turn + kRing);
  }
}

template <typename T, int VEC, int NV, int GROUP, int U, bool MX, bool FULL>
__global__ void __launch_bounds__(kThreads, NV * VEC * sizeof(T) <= 32 ? 2 : 1)
    ln_bwd_stream_kernel(const T* __restrict__ dy, const T* __restrict__ x, const uint8_t* __restrict__ codes,
                         const uint8_t* __restrict__ scales, const float* __restrict__ mean_in,
                         const float* __restrict__ rstd_in, const float* __restrict__ gamma,
                         const T* __restrict__ residual, T* __restrict__ dx, float* __restrict__ dgamma,
                         float* __restrict__ dbeta, int64_t partial_stride, int64_t rows, int c, int* err) {
  constexpr int kTeam = GROUP <= 32 ? 32 : kThreads;
  constexpr int kGroups = kTeam / GROUP;
  constexpr int RS = kGroups * U;
  using Codes = typename MxCodes<VEC>::type;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint64_t bars[kThreads / kTeam * kRing];
  __shared__ float scratch[4 * U * kWarps];
  int turn_of = 0;
  const int t = threadIdx.x % GROUP, g = threadIdx.x % kTeam / GROUP;
  const bool leader = threadIdx.x % kTeam == 0;
  const int blocks = (c + kMxBlock - 1) / kMxBlock;
  const float inv_c = 1.0f / static_cast<float>(c);
  Ring<kTeam, RS> ring(smem, bars, rows);
  ring.add(dy, c * static_cast<int>(sizeof(T)));
  if constexpr (MX)
    ring.add(codes, c);
  else
    ring.add(x, c * static_cast<int>(sizeof(T)));
  if (residual != nullptr) ring.add(residual, c * static_cast<int>(sizeof(T)));
  ring.place();
  __syncthreads();
  if (leader)
    for (int i = 0; i < kRing; ++i) ring.fetch(i);
  Lanes<VEC> dg[NV], db[NV], w[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int col = (i * GROUP + t) * VEC;
    dg[i] = db[i] = Lanes<VEC>(0.f);
    w[i] = (FULL || col < c) && gamma != nullptr ? load_weight<VEC>(gamma + col) : Lanes<VEC>(1.f);
  }
  // a chunk's statistics (and scales) are loaded while the one before it is worked on
  float mean[U], rstd[U];
  uint8_t scale[MX ? U : 1][NV];
  auto load_statistics = [&](int64_t row0) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t row = row0 + g + u * kGroups;
      const bool in = row < rows;
      mean[u] = in ? __ldg(mean_in + row) : 0.f;
      rstd[u] = in ? __ldg(rstd_in + row) : 0.f;
      if constexpr (MX) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int col = (i * GROUP + t) * VEC;
          scale[u][i] = in && (FULL || col < c) ? __ldg(scales + row * blocks + col / kMxBlock) : 0;
        }
      }
    }
  };
  load_statistics(ring.row(0));
  for (int turn = 0; ring.row(turn) < rows; ++turn) {
    float m[U], r[U], scaled[MX ? U : 1][NV];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      m[u] = -mean[u];
      r[u] = rstd[u];
      if constexpr (MX)
#pragma unroll
        for (int i = 0; i < NV; ++i) scaled[u][i] = mx_scale(scale[u][i]);
    }
    load_statistics(ring.row(turn + 1));
    if (!ring.wait(turn, err)) break;
    const int64_t row0 = ring.row(turn) + g;
    const T* have_dy = ring.template at<T>(turn, 0) + g * c;
    const uint8_t* have_x = ring.template at<uint8_t>(turn, RS * c * static_cast<int>(sizeof(T)));
    const T* have_res = ring.template at<T>(turn, RS * c * static_cast<int>(sizeof(T) + (MX ? 1 : sizeof(T)))) + g * c;
    const bool whole = ring.row(turn) + RS <= rows;  // the same for the team
    // dy and the normalised input of row u, vector i; 0 for a row past the last one (the slot holds what was
    // there before). The mean is taken off first: x rstd - mean rstd would leave rounding errors of mean
    // rstd where a row hardly varies. Where dy is 0 (past a row's end) no sum sees xh.
    auto read = [&](int u, int i, Lanes<VEC>& d, Lanes<VEC>& xh) {
      const int col = (i * GROUP + t) * VEC;
      const int at = u * kGroups * c + col;
      d = widen<T, VEC>(FULL || col < c ? shared_raw<T, VEC>(have_dy + at) : zero_raw<T, VEC>());
      if constexpr (MX) {
        const Codes q = FULL || col < c ? *reinterpret_cast<const Codes*>(have_x + g * c + at) : Codes{};
        xh = fma(mx_codes_value<VEC>(q), Lanes<VEC>(scaled[u][i]), Lanes<VEC>(m[u])) * Lanes<VEC>(r[u]);
      } else {
        xh = (widen<T, VEC>(FULL || col < c ? shared_raw<T, VEC>(reinterpret_cast<const T*>(have_x) + g * c + at)
                                            : zero_raw<T, VEC>()) +
              Lanes<VEC>(m[u])) *
             Lanes<VEC>(r[u]);
      }
      if (!whole && row0 + u * kGroups >= rows) d = xh = Lanes<VEC>(0.f);
    };
    // dgamma, dbeta and the row's sums; d becomes gamma dy
    auto add = [&](int i, Lanes<VEC>& d, const Lanes<VEC>& xh, float& s0, float& s1) {
      dg[i] = fma(d, xh, dg[i]);
      db[i] = db[i] + d;
      d = d * w[i];
      s0 += d.sum();
      s1 += d.dot(xh);
    };
    // dx = rstd w - rstd mean(w) - xh rstd mean(w xh)
    auto finish = [&](int u, int i, const Lanes<VEC>& d, const Lanes<VEC>& xh, float s0, float s1) {
      const int64_t row = row0 + u * kGroups;
      const int col = (i * GROUP + t) * VEC;
      if (row < rows && (FULL || col < c)) {
        Lanes<VEC> o = fma(xh, Lanes<VEC>(-s1 * inv_c * r[u]), fma(d, Lanes<VEC>(r[u]), Lanes<VEC>(-s0 * inv_c * r[u])));
        if (residual != nullptr) o = o + widen<T, VEC>(shared_raw<T, VEC>(have_res + u * kGroups * c + col));
        store_lanes<T, VEC>(dx + row * c + col, o);
      }
    };
    if constexpr (GROUP > 32) {
      // the block's barriers cost more than reading the slot again: all rows of the chunk at a time
      float s[2 * U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        s[2 * u] = s[2 * u + 1] = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          Lanes<VEC> d, xh;
          read(u, i, d, xh);
          add(i, d, xh, s[2 * u], s[2 * u + 1]);
        }
      }
      group_sum<GROUP>(s, scratch, turn_of);
#pragma unroll
      for (int u = 0; u < U; ++u) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          Lanes<VEC> d, xh;
          read(u, i, d, xh);
          finish(u, i, d * w[i], xh, s[2 * u], s[2 * u + 1]);
        }
      }
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        Lanes<VEC> xh[NV], d[NV];
        float s[2] = {0.f, 0.f};
#pragma unroll
        for (int i = 0; i < NV; ++i) read(u, i, d[i], xh[i]);
#pragma unroll
        for (int i = 0; i < NV; ++i) add(i, d[i], xh[i], s[0], s[1]);
        group_sum<GROUP>(s, scratch, turn_of);
#pragma unroll
        for (int i = 0; i < NV; ++i) finish(u, i, d[i], xh[i], s[0], s[1]);
      }
    }
    team_sync<kTeam>();
    if (leader) ring.fetch(turn + kRing);
  }
  // the rings hold 24 rows or more, at least 72 bytes a channel: room for 32 bytes a lane's channel, of which at
  // most half lie past the row
  write_column_sums<VEC, NV, GROUP>(dg, db, dgamma, dbeta, partial_stride, c, reinterpret_cast<float*>(smem));
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
    uint32_t byte;
    const auto q = mx_quantise<T, VEC>(v[u], widen<T, VEC>(v[u]), byte);
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
    if (p.in) store_lanes<T, VEC>(x + p.at, mx_codes_value<VEC>(v[u]) * Lanes<VEC>(mx_scale(s[u])));
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
    const Lanes<VEC> a = widen<T, VEC>(va[u]), b = widen<T, VEC>(vb[u]);
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
    if (in)
      store_lanes<T, VEC>(out + static_cast<int64_t>(id) * VEC, a.each([](float v) {
                            const Gate g(v);
                            return v * g.f * g.u;
                          }) * b);
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
    const Lanes<VEC> d = widen<T, VEC>(vd[u]);
    Lanes<VEC> a, b;
    if constexpr (MX) {
      a = mx_codes_value<VEC>(ca[u]) * Lanes<VEC>(mx_scale(sa[u]));
      b = mx_codes_value<VEC>(cb[u]) * Lanes<VEC>(mx_scale(sb[u]));
    } else {
      a = widen<T, VEC>(va[u]);
      b = widen<T, VEC>(vb[u]);
    }
    const Lanes<VEC> unit = a.each([](float v) {
      const Gate g(v);
      return v * g.f * g.u;
    });
    // the gate's factors one at a time: d b f first, so that a large 1 + a (1 - s) meets it when it is small
    Lanes<VEC> da = d * b;
    da = a.apply(da, [](float v, float w) {
      const Gate g(v);
      return w * g.f * (1.0f + v * g.c) * g.u;
    });
    store_lanes<T, VEC>(dab + at[u], da);
    store_lanes<T, VEC>(dab + at[u] + h, d * unit);
    if (out != nullptr) store_lanes<T, VEC>(out + static_cast<int64_t>(id) * VEC, unit * b);
  }
}

// ------------------------------------------------------------------ launches
bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

#define FFB_ROW(V, N, G, U)                                                                                   \
  if (c <= (V) * (N) * (G))                                                                                   \
  return f(std::integral_constant<int, V>{}, std::integral_constant<int, N>{}, std::integral_constant<int, G>{}, \
           std::integral_constant<int, U>{})

// How a row of c channels is held, for rows that are streamed: vectors of 16 bytes, two a thread where the
// row allows it (fewer threads, fewer shuffles to add them up; more would leave few registers), and U rows
// of a group at a time so that a chunk is a few KB. Calls f(VEC, NV, GROUP, U as integral constants).
template <typename T, typename F>
int dispatch_stream(int c, F&& f) {
  constexpr int kVec = 16 / sizeof(T);
  if constexpr (kVec == 8) {
    FFB_ROW(8, 2, 4, 2);
    FFB_ROW(8, 2, 8, 2);
    FFB_ROW(8, 2, 16, 2);
    FFB_ROW(8, 2, 32, 2);
    FFB_ROW(8, 4, 32, 1);
    FFB_ROW(8, 2, kThreads, 2);
    FFB_ROW(8, 4, kThreads, 1);
  } else {
    FFB_ROW(4, 2, 8, 2);
    FFB_ROW(4, 2, 16, 2);
    FFB_ROW(4, 2, 32, 2);
    FFB_ROW(4, 4, 32, 1);
    FFB_ROW(4, 2, kThreads, 2);
    FFB_ROW(4, 4, kThreads, 1);
    FFB_ROW(4, 8, kThreads, 1);
  }
  return static_cast<int>(cudaErrorInvalidValue);
}

// The same for rows that are not: vectors where every pointer is 16-byte aligned and c a whole number of
// them, else single elements; the fewest threads that hold a row with at most 32 channels a thread.
template <typename T, typename F>
int dispatch_row(int c, bool vector, F&& f) {
  constexpr int kVec = 16 / sizeof(T);
  if (vector) {
    FFB_ROW(kVec, 1, 32, 2);
    FFB_ROW(kVec, 32 / kVec, 32, 1);
    FFB_ROW(kVec, 32 / kVec, kThreads, 1);
  } else {
    FFB_ROW(1, 2, 32, 4);
    FFB_ROW(1, 8, 32, 2);
    FFB_ROW(1, 8, kThreads, 2);
    FFB_ROW(1, 32, kThreads, 1);
  }
  return static_cast<int>(cudaErrorInvalidValue);
}
#undef FFB_ROW

constexpr int kLnBlocks = 148 * 2;  // blocks (rows of partial sums) of the backward pass at most

// Whether rows of c channels are streamed: 16-byte words (every pointer is aligned) of 16 channels, and a
// block's rings, whose rows take `row_bytes` over all tensors, fit shared memory (fp32 rows of above 6000
// channels with a residual do not).
template <typename T>
bool ln_streams(bool whole, int c, int row_bytes) {
  int per = 0;
  dispatch_stream<T>(c, [&](auto, auto, auto g, auto u) {
    per = kThreads / decltype(g)::value * decltype(u)::value;
    return 0;
  });
  return whole && c % 16 == 0 && static_cast<int64_t>(kRing) * per * row_bytes <= 200 * 1024;
}

// blocks of a backward pass whose blocks take `per` rows at a time
int ln_blocks(int64_t rows, int64_t per) {
  const int64_t want = (rows + per - 1) / per;
  return static_cast<int>(want < kLnBlocks ? want : kLnBlocks);
}
template <typename T>
int ln_bwd_blocks(int64_t rows, int c, bool stream, bool vector) {
  int blocks = 0;
  auto count = [&](auto, auto, auto g, auto u) {
    blocks = ln_blocks(rows, kThreads / decltype(g)::value * decltype(u)::value);
    return 0;
  };
  if (stream)
    dispatch_stream<T>(c, count);
  else
    dispatch_row<T>(c, vector, count);
  return blocks;
}

template <typename T>
int ln_train(const LayerNormTrain& p, int* err, cudaStream_t stream) {
  const bool whole = aligned(p.x) && aligned(p.y) && aligned(p.codes) && aligned(p.gamma) && aligned(p.beta);
  if (ln_streams<T>(whole, p.c, p.c * sizeof(T)))
    return dispatch_stream<T>(p.c, [&](auto v, auto n, auto g, auto u) {
      constexpr int V = decltype(v)::value, N = decltype(n)::value, G = decltype(g)::value, U = decltype(u)::value;
      constexpr int per = kThreads / G * U;  // rows of a block at a time
      auto kernel = p.c == V * N * G ? ln_train_stream_kernel<T, V, N, G, U, true> : ln_train_stream_kernel<T, V, N, G, U, false>;
      const int smem = kRing * per * p.c * static_cast<int>(sizeof(T));
      const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
      if (e != cudaSuccess) return static_cast<int>(e);
      kernel<<<ln_blocks(p.rows, per), kThreads, smem, stream>>>(static_cast<const T*>(p.x), static_cast<T*>(p.y), p.gamma,
                                                                p.beta, p.mean, p.rstd, p.codes, p.scales, p.rows, p.c,
                                                                p.eps, err);
      return static_cast<int>(cudaGetLastError());
    });
  return dispatch_row<T>(p.c, whole && p.c % (16 / sizeof(T)) == 0, [&](auto v, auto n, auto g, auto u) {
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
int ln_bwd(const LayerNormBwd& p, int* err, cudaStream_t stream) {
  const bool mx = p.codes != nullptr;
  const bool whole = aligned(p.dy) && aligned(p.dx) && aligned(p.residual) && aligned(p.gamma) &&
                     aligned(mx ? static_cast<const void*>(p.codes) : p.x);
  const int row_bytes = p.c * static_cast<int>(sizeof(T)), all_bytes = row_bytes + (mx ? p.c : row_bytes) + (p.residual != nullptr ? row_bytes : 0);
  const bool streamed = ln_streams<T>(whole, p.c, all_bytes), vector = whole && p.c % (16 / sizeof(T)) == 0;
  const int grid = ln_bwd_blocks<T>(p.rows, p.c, streamed, vector);
  const bool sums = p.dgamma != nullptr || p.dbeta != nullptr;
  // one block writes the gradients itself; several leave rows [dgamma | dbeta] of partial sums
  float* part = static_cast<float*>(p.workspace);
  float* dg = !sums ? nullptr : grid == 1 ? p.dgamma : part;
  float* db = !sums ? nullptr : grid == 1 ? p.dbeta : part + p.c;
  const int64_t stride = 2 * static_cast<int64_t>(p.c);
  const T* dy = static_cast<const T*>(p.dy);
  const T* x = static_cast<const T*>(p.x);
  const T* residual = static_cast<const T*>(p.residual);
  T* dx = static_cast<T*>(p.dx);
  int rc;
  if (streamed)
    rc = dispatch_stream<T>(p.c, [&](auto v, auto n, auto g, auto u) {
      constexpr int V = decltype(v)::value, N = decltype(n)::value, G = decltype(g)::value, U = decltype(u)::value;
      constexpr int per = kThreads / G * U;
      const int smem = kRing * per * all_bytes;
      const bool full = p.c == V * N * G;
      auto kernel = mx ? full ? ln_bwd_stream_kernel<T, V, N, G, U, true, true> : ln_bwd_stream_kernel<T, V, N, G, U, true, false>
                       : full ? ln_bwd_stream_kernel<T, V, N, G, U, false, true> : ln_bwd_stream_kernel<T, V, N, G, U, false, false>;
      const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
      if (e != cudaSuccess) return static_cast<int>(e);
      kernel<<<grid, kThreads, smem, stream>>>(dy, x, p.codes, p.scales, p.mean, p.rstd, p.gamma, residual, dx, dg, db,
                                               stride, p.rows, p.c, err);
      return static_cast<int>(cudaGetLastError());
    });
  else
    rc = dispatch_row<T>(p.c, vector, [&](auto v, auto n, auto g, auto u) {
      constexpr int V = decltype(v)::value, N = decltype(n)::value, G = decltype(g)::value, U = decltype(u)::value;
      auto kernel = mx ? ln_bwd_kernel<T, V, N, G, U, true> : ln_bwd_kernel<T, V, N, G, U, false>;
      kernel<<<grid, kThreads, 0, stream>>>(dy, x, p.codes, p.scales, p.mean, p.rstd, p.gamma, residual, dx, dg, db, stride,
                                            p.rows, p.c);
      return static_cast<int>(cudaGetLastError());
    });
  if (rc == 0 && sums && grid > 1) {
    ln_grad_reduce_kernel<<<(2 * p.c + 31) / 32, 1024, 0, stream>>>(part, p.dgamma, p.dbeta, grid, p.c);
    rc = static_cast<int>(cudaGetLastError());
  }
  return rc;
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
  // the tensors' alignment is not known here: room for the form with the most blocks
  int most = 0;
  for (int form = 0; form < 3; ++form) {
    const bool stream = form == 0, vector = form == 1;
    const int blocks = is_f32 ? ln_bwd_blocks<float>(rows, c, stream, vector) : ln_bwd_blocks<__nv_bfloat16>(rows, c, stream, vector);
    if (blocks > most) most = blocks;
  }
  return most > 1 ? static_cast<size_t>(most) * 2 * c * sizeof(float) : 0;
}

int launch_ln_train(const LayerNormTrain& p, int is_f32, int* err, cudaStream_t stream) {
  return is_f32 ? ln_train<float>(p, err, stream) : ln_train<__nv_bfloat16>(p, err, stream);
}
int launch_ln_bwd(const LayerNormBwd& p, int is_f32, int* err, cudaStream_t stream) {
  return is_f32 ? ln_bwd<float>(p, err, stream) : ln_bwd<__nv_bfloat16>(p, err, stream);
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
