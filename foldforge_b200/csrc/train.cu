// Training operators bound by memory: LayerNorm forward and backward, the 8-bit checkpoint
// (mx8.cuh) packed and read back, and the gated unit silu(a) b forward and backward.
//
// Measured on one B200 (device time, L2 holding other data; a plain copy moves 6.5 TB/s):
//   LayerNorm, 262144 x 128 bf16 (a pair tensor of 512 tokens)   forward 21 us (6.4 TB/s), writing a
//     checkpoint too 29 us (5.8); backward 36 us (5.6), from a checkpoint 37 us (4.6), and 4 us for the sums
//     over the blocks. With rows loaded straight to registers instead of rings the four took 32 / 43 / 45 / 50 us:
//     what was in flight was limited by the registers, at 16 warps an SM. With a checkpoint, work on the
//     values weighs as well: 59 and 62% of issue slots in a profile of these two, the memory's pins at 46 and 41%.
//     (The backward pass from a checkpoint has 4 to 8 bytes of a thread's registers spilled where rows are
//     full, the forward pass of 1025 to 4096 channels in whole blocks of 16 bytes 16 to 40.)
//   LayerNorm, 4099 x 4096 bf16 with a checkpoint   19 us + 25 us + 4 us
//   checkpoint, 524288 x 64 bf16   packed in 15 us, read back in 12 us
//   gated unit, 65536 x 2 x 512 bf16 with a checkpoint   49 us (5.5 TB/s), backward 50 us (4.1)
#include <initializer_list>
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

// The sum of N (a power of two) values as a tree, in which equal values add up without rounding.
template <int N>
__device__ __forceinline__ float tree_sum(float (&v)[N]) {
#pragma unroll
  for (int n = N / 2; n > 0; n /= 2)
#pragma unroll
    for (int i = 0; i < n; ++i) v[i] += v[i + n];
  return v[0];
}

// Sums `v` over the GROUP threads that share a row (4 to 32, or the whole block). The block form
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
      float w[kWarps];
#pragma unroll
      for (int i = 0; i < kWarps; ++i) w[i] = s[k * kWarps + i];
      v[k] = tree_sum(w);
    }
  }
}

// ------------------------------------------------------------------ LayerNorm
// VEC sums to fp32 memory of any alignment
template <int VEC>
__device__ __forceinline__ void store_sums(float* p, const Lanes<VEC>& v) {
  if (VEC > 1 && (reinterpret_cast<uintptr_t>(p) & 15u) == 0) {
#pragma unroll
    for (int j = 0; j + 4 <= VEC; j += 4)
      *reinterpret_cast<float4*>(p + j) = make_float4(v.get(j), v.get(j + 1), v.get(j + 2), v.get(j + 3));
  } else {
#pragma unroll
    for (int j = 0; j < VEC; ++j) p[j] = v.get(j);
  }
}

// The block's sums of each channel over its rows (dg, db: a thread's, over the rows it took) to row
// blockIdx.x of the partial sums. `space` holds kWarps NV GROUP VEC floats unless the whole block shares
// each row, and nobody uses it any more once the block has come here.
template <int VEC, int NV, int GROUP>
__device__ __forceinline__ void write_column_sums(Lanes<VEC> (&dg)[NV], Lanes<VEC> (&db)[NV], float* dgamma, float* dbeta,
                                                  int64_t partial_stride, int c, float* space) {
  if (dgamma == nullptr && dbeta == nullptr) return;
  let_next_kernel_start();
  const int t = threadIdx.x % GROUP;
  float* pg = dgamma == nullptr ? nullptr : dgamma + blockIdx.x * partial_stride;
  float* pb = dbeta == nullptr ? nullptr : dbeta + blockIdx.x * partial_stride;
  if constexpr (GROUP == kThreads) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int col = (i * GROUP + t) * VEC;
      if (col < c && pg != nullptr) store_sums<VEC>(pg + col, dg[i]);
      if (col < c && pb != nullptr) store_sums<VEC>(pb + col, db[i]);
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

// Rows are streamed: a team (a warp, or the block for rows that a warp's registers cannot hold) takes RS
// rows at a time, which lie next to one another in memory, and has them copied to its own ring of slots in
// shared memory by bulk copies. The loads in flight then do not depend on registers or occupancy, and cost
// one thread a few instructions.
constexpr int kRing = 3;  // slots at most

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

// bytes of a slot for `rows` rows of a tensor: they start at any of 16 bytes, and whole granules are copied
__host__ __device__ constexpr int slot_part(int rows, int row_bytes) { return (rows * row_bytes + 30) / 16 * 16; }

// A team's ring over `streams` tensors (16-byte aligned, rows of row_bytes[k] bytes); a slot holds RS rows of
// each, one tensor after the other. WHOLE: rows are whole 16-byte granules in every tensor. Otherwise the
// copies take the aligned granules around the rows, and the tensor's last bytes, where they do not fill one,
// are written by the copying thread itself.
template <int TEAM, int RS, bool WHOLE>
struct Ring {
  uint8_t* slots;
  uint64_t* full;
  int depth, slot, phase;  // slots, the one in use and the parity its next copies complete
  int streams, slot_bytes;
  const uint8_t* base[3];
  int row_bytes[3];
  int64_t rows, teams, first;  // this team's chunks of RS rows: first, first + teams, ..

  __device__ __forceinline__ Ring(uint8_t* smem, uint64_t* bars, int slots_of, int64_t all_rows)
      : depth(slots_of), slot(0), phase(0), streams(0), slot_bytes(0), rows(all_rows) {
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
    slot_bytes += part(bytes);
    ++streams;
  }
  __device__ __forceinline__ static int part(int bytes) { return WHOLE ? RS * bytes : slot_part(RS, bytes); }
  // after the last add: the team's part of shared memory
  __device__ __forceinline__ void place() { slots += static_cast<int64_t>(threadIdx.x / TEAM) * depth * slot_bytes; }
  __device__ __forceinline__ int64_t row(int turn) const { return (first + turn * teams) * RS; }
  // one thread: the copies of the team's chunk number `turn` into slot `to`
  __device__ __forceinline__ void fetch(int turn, int to) {
    const int64_t at = row(turn);
    if (at >= rows) return;
    const int n = rows - at < RS ? static_cast<int>(rows - at) : RS;
    uint64_t* bar = &full[to];
    uint8_t* dst = slots + to * slot_bytes;
    if constexpr (WHOLE) {
      int all = 0;
#pragma unroll
      for (int k = 0; k < 3; ++k)
        if (k < streams) all += n * row_bytes[k];
      mbar_arrive_expect_tx(bar, all);
#pragma unroll
      for (int k = 0; k < 3; ++k)
        if (k < streams) {
          bulk_load(dst, base[k] + at * row_bytes[k], n * row_bytes[k], bar);
          dst += RS * row_bytes[k];
        }
      return;
    }
    uint32_t bytes[3] = {0, 0, 0}, all = 0;
#pragma unroll
    for (int k = 0; k < 3; ++k)
      if (k < streams) {
        const uint8_t* a = base[k] + at * row_bytes[k];
        const uint8_t* stop = a + n * row_bytes[k];
        const uint8_t* from = a - (reinterpret_cast<uintptr_t>(a) & 15u);
        const uint8_t* end = base[k] + rows * row_bytes[k];
        const uint8_t* whole = end - (reinterpret_cast<uintptr_t>(end) & 15u);  // granules past here are not the tensor's alone
        const uint8_t* to_here = stop + ((16u - (reinterpret_cast<uintptr_t>(stop) & 15u)) & 15u);
        if (to_here > whole) to_here = whole;
        for (const uint8_t* q = to_here > from ? to_here : from; q < stop; ++q) dst[q - from] = __ldg(q);
        bytes[k] = to_here > from ? static_cast<uint32_t>(to_here - from) : 0u;
        all += bytes[k];
        dst += slot_part(RS, row_bytes[k]);
      }
    mbar_arrive_expect_tx(bar, all);
    dst = slots + to * slot_bytes;
#pragma unroll
    for (int k = 0; k < 3; ++k)
      if (k < streams) {
        const uint8_t* a = base[k] + at * row_bytes[k];
        if (bytes[k] != 0) bulk_load(dst, a - (reinterpret_cast<uintptr_t>(a) & 15u), bytes[k], bar);
        dst += slot_part(RS, row_bytes[k]);
      }
  }
  __device__ __forceinline__ void start() {
    for (int i = 0; i < depth; ++i) fetch(i, i);
  }
  // False (for the whole team) where the copies never came: the error word says so, and the other slots'
  // copies have had the same time to land.
  __device__ __forceinline__ bool wait(int* err) {
    return team_all<TEAM>(mbar_wait(&full[slot], phase, err, kErrTimeoutLoad));
  }
  // the team has read chunk `turn`: its slot takes a later one
  __device__ __forceinline__ void next(int turn) {
    team_sync<TEAM>();
    if (threadIdx.x % TEAM == 0) fetch(turn + depth, slot);
    if (++slot == depth) {
      slot = 0;
      phase ^= 1;
    }
  }
  // the first row of chunk `turn` in tensor k, whose part of a slot starts at `offset`
  template <typename P>
  __device__ __forceinline__ const P* at(int turn, int k, int offset) const {
    const uint32_t shift = WHOLE ? 0 : static_cast<uint32_t>(reinterpret_cast<uintptr_t>(base[k] + row(turn) * row_bytes[k])) & 15u;
    return reinterpret_cast<const P*>(slots + slot * slot_bytes + offset + shift);
  }
};

// ROWS says what is known of a row. kFullRows: c fills the group's vectors, so that no lane has to look
// whether its channels are there; kWholeRows: c is a multiple of 16; kAnyRows: nothing.
enum Rows : int { kAnyRows, kWholeRows, kFullRows };

// ---- forward. GROUP threads hold a row in registers (NV vectors of VEC channels a thread): mean and variance
// in two passes over the registers, one read and one write an element. Writes each row's mean and
// 1 / sqrt(var + eps) in fp32 for the backward pass and, with `codes`, the input's 8-bit checkpoint.
template <typename T, int VEC, int NV, int GROUP, int U, Rows ROWS>
__global__ void __launch_bounds__(kThreads, NV * VEC * sizeof(T) <= 32 ? 2 : 1)
    ln_train_kernel(const T* __restrict__ x, T* __restrict__ y, const float* __restrict__ gamma,
                    const float* __restrict__ beta, float* __restrict__ mean_out, float* __restrict__ rstd_out,
                    uint8_t* __restrict__ codes, uint8_t* __restrict__ scales, int64_t rows, int c, float eps, int slots,
                    int* err) {
  constexpr bool FULL = ROWS == kFullRows;
  constexpr int kTeam = GROUP <= 32 ? 32 : kThreads;
  constexpr int kGroups = kTeam / GROUP;  // rows of a team side by side
  constexpr int RS = kGroups * U;
  constexpr int kLanes = kMxBlock / VEC;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint64_t bars[kThreads / kTeam * kRing];
  __shared__ float scratch[2 * U * kWarps];
  int turn_of = 0;
  const int t = threadIdx.x % GROUP, g = threadIdx.x % kTeam / GROUP;
  const int blocks = (c + kMxBlock - 1) / kMxBlock;
  const float inv_c = 1.0f / static_cast<float>(c);
  Ring<kTeam, RS, (ROWS > 0)> ring(smem, bars, slots, rows);
  ring.add(x, c * static_cast<int>(sizeof(T)));
  ring.place();
  __syncthreads();
  if (threadIdx.x % kTeam == 0) ring.start();
  Lanes<VEC> w[NV], b[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int col = (i * GROUP + t) * VEC;
    w[i] = (FULL || col < c) && gamma != nullptr ? load_weight<VEC>(gamma + col) : Lanes<VEC>(1.f);
    b[i] = (FULL || col < c) && beta != nullptr ? load_weight<VEC>(beta + col) : Lanes<VEC>(0.f);
  }
  for (int turn = 0; ring.row(turn) < rows; ++turn) {
    if (!ring.wait(err)) break;
    const int64_t row0 = ring.row(turn) + g;
    const T* have = ring.template at<T>(turn, 0, 0) + g * c;
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
    auto finish = [&](const typename Raw<T, VEC>::type (&v)[NV], const Lanes<VEC> (&f)[NV], float m, float r, int64_t row) {
      if (codes != nullptr) {
        typename MxCodes<VEC>::type q[NV];
        uint32_t byte[NV];
        mx_quantise<T, VEC, NV>(v, f, q, byte);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int col = (i * GROUP + t) * VEC;
          if (row < rows && (FULL || col < c)) {
            *reinterpret_cast<typename MxCodes<VEC>::type*>(codes + row * c + col) = q[i];
            if (t % kLanes == 0) scales[row * blocks + col / kMxBlock] = static_cast<uint8_t>(byte[i]);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int col = (i * GROUP + t) * VEC;
        if (row < rows && (FULL || col < c))
          store_lanes<T, VEC>(y + row * c + col, fma((f[i] + Lanes<VEC>(-m)) * Lanes<VEC>(r), w[i], b[i]));
      }
    };
    auto keep = [&](float m, float r, int64_t row) {
      if (t == 0 && row < rows) {
        mean_out[row] = m;
        rstd_out[row] = r;
      }
    };
    // rows of a block together: a barrier for all of them
    constexpr int kTogether = GROUP > 32 ? U : 1;
#pragma unroll
    for (int u0 = 0; u0 < U; u0 += kTogether) {
      typename Raw<T, VEC>::type v[kTogether][NV];
      Lanes<VEC> f[kTogether][NV];
      // The mean of a row that does not vary is its value to the last bit: the sums are trees, in which equal
      // values add up without rounding, and that is all there is to a full row (c is a power of two). Of
      // other rows each vector's sum, or that of two single elements, has the first channel taken off as often
      // as it holds it, before 3 or 5 of them add up. For 65536 x 384 bf16 that costs 0.6 us of 21.6; taking it
      // off every element of every row 1.3.
      float m[kTogether], r[kTogether], x0[kTogether];
#pragma unroll
      for (int u = 0; u < kTogether; ++u) {
        constexpr int kSum = VEC > 1 ? 1 : 2;  // of NV vectors
        float sums[NV / kSum];
        x0[u] = FULL ? 0.f : static_cast<float>(have[(u0 + u) * kGroups * c]);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          v[u][i] = read(u0 + u, i);
          f[u][i] = widen<T, VEC>(v[u][i]);
        }
#pragma unroll
        for (int i = 0; i < NV; i += kSum) {
          const int col = (i * GROUP + t) * VEC;
          float a = f[u][i].tree();
          if constexpr (kSum == 2) a += f[u][i + 1].tree();
          if constexpr (!FULL) a = col < c ? fmaf(kSum == 2 && col + GROUP < c ? -2.f : -static_cast<float>(VEC), x0[u], a) : 0.f;
          sums[i / kSum] = a;
        }
        m[u] = tree_sum(sums);
      }
      group_sum<GROUP>(m, scratch, turn_of);
#pragma unroll
      for (int u = 0; u < kTogether; ++u) {
        m[u] = fmaf(m[u], inv_c, x0[u]);
        r[u] = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) r[u] += squares(f[u][i], m[u], i);
      }
      group_sum<GROUP>(r, scratch, turn_of);
#pragma unroll
      for (int u = 0; u < kTogether; ++u) {
        const int64_t row = row0 + (u0 + u) * kGroups;
        r[u] = rsqrtf(r[u] * inv_c + eps);
        keep(m[u], r[u], row);
        finish(v[u], f[u], m[u], r[u], row);
      }
    }
    ring.next(turn);
  }
}

// ---- backward. xh = (x - mean) rstd, w = gamma dy: dx = rstd (w - mean(w) - xh mean(w xh)) (+ residual). A
// thread keeps the same channels for every row it takes, so the sums dgamma = sum dy xh and dbeta = sum dy
// stay in its registers until the end; the block's row groups are then added in a fixed order and each
// block writes one row of partial sums, which ln_grad_reduce_kernel adds in a fixed order: the result does
// not depend on timing.
template <typename T, int VEC, int NV, int GROUP, int U, bool MX, Rows ROWS>
__global__ void __launch_bounds__(kThreads, NV * VEC * sizeof(T) <= 32 ? 2 : 1)
    ln_bwd_kernel(const T* __restrict__ dy, const T* __restrict__ x, const uint8_t* __restrict__ codes,
                  const uint8_t* __restrict__ scales, const float* __restrict__ mean_in,
                  const float* __restrict__ rstd_in, const float* __restrict__ gamma, const T* __restrict__ residual,
                  T* __restrict__ dx, float* __restrict__ dgamma, float* __restrict__ dbeta, int64_t partial_stride,
                  int64_t rows, int c, int slots, int* err) {
  constexpr bool FULL = ROWS == kFullRows;
  constexpr int kTeam = GROUP <= 32 ? 32 : kThreads;
  constexpr int kGroups = kTeam / GROUP;
  constexpr int RS = kGroups * U;
  using Codes = typename MxCodes<VEC>::type;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint64_t bars[kThreads / kTeam * kRing];
  __shared__ float scratch[4 * U * kWarps];
  int turn_of = 0;
  const int t = threadIdx.x % GROUP, g = threadIdx.x % kTeam / GROUP;
  const int blocks = (c + kMxBlock - 1) / kMxBlock;
  const float inv_c = 1.0f / static_cast<float>(c);
  Ring<kTeam, RS, (ROWS > 0)> ring(smem, bars, slots, rows);
  ring.add(dy, c * static_cast<int>(sizeof(T)));
  if constexpr (MX)
    ring.add(codes, c);
  else
    ring.add(x, c * static_cast<int>(sizeof(T)));
  if (residual != nullptr) ring.add(residual, c * static_cast<int>(sizeof(T)));
  ring.place();
  __syncthreads();
  if (threadIdx.x % kTeam == 0) ring.start();
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
    if (!ring.wait(err)) break;
    const int64_t row0 = ring.row(turn) + g;
    const int row_bytes = c * static_cast<int>(sizeof(T)), part = ring.part(row_bytes);
    const T* have_dy = ring.template at<T>(turn, 0, 0) + g * c;
    const uint8_t* have_x = ring.template at<uint8_t>(turn, 1, part);
    const T* have_res = residual == nullptr ? nullptr : ring.template at<T>(turn, 2, part + ring.part(MX ? c : row_bytes)) + g * c;
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
    ring.next(turn);
  }
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
  wait_for_kernel_before();
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
  Lanes<VEC> f[U];
  typename MxCodes<VEC>::type q[U];
  uint32_t byte[U];
#pragma unroll
  for (int u = 0; u < U; ++u) f[u] = widen<T, VEC>(v[u]);
  mx_quantise<T, VEC, U>(v, f, q, byte);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const P p(first + u * kThreads, total, c, per_row);
    if (p.in) {
      *reinterpret_cast<typename MxCodes<VEC>::type*>(codes + p.at) = q[u];
      if (threadIdx.x % P::kLanes == 0) scales[p.block] = static_cast<uint8_t>(byte[u]);
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
    const typename Raw<T, VEC>::type v[2] = {va[u], vb[u]};
    const Lanes<VEC> f[2] = {widen<T, VEC>(va[u]), widen<T, VEC>(vb[u])};
    const Lanes<VEC>&a = f[0], &b = f[1];
    if (codes != nullptr) {
      typename MxCodes<VEC>::type q[2];
      uint32_t byte[2];
      mx_quantise<T, VEC, 2>(v, f, q, byte);
      if (in) {
        *reinterpret_cast<typename MxCodes<VEC>::type*>(codes + at[u]) = q[0];
        *reinterpret_cast<typename MxCodes<VEC>::type*>(codes + at[u] + h) = q[1];
        if (threadIdx.x % kLanes == 0) {  // whole blocks: the scales of a row are 2 h / 32
          uint8_t* s = scales + at[u] / kMxBlock;
          s[0] = static_cast<uint8_t>(byte[0]);
          s[h / kMxBlock] = static_cast<uint8_t>(byte[1]);
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

// How a row of c channels is held: vectors of 16 bytes where it is a whole number of them, two a thread
// where the row allows it (fewer threads, fewer shuffles to add them up; more would leave few registers),
// else single elements, 32 lanes side by side; and U rows of a group at a time so that a chunk is a few KB.
// Calls f(VEC, NV, GROUP, U as integral constants).
template <typename T, typename F>
int dispatch_row(int c, F&& f) {
  constexpr int kVec = 16 / sizeof(T);
  if (c % kVec != 0) {
    FFB_ROW(1, 2, 32, 4);
    FFB_ROW(1, 8, 32, 2);
    FFB_ROW(1, 32, 32, 1);
    FFB_ROW(1, 8, kThreads, 2);
    FFB_ROW(1, 32, kThreads, 1);
  } else if constexpr (kVec == 8) {
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
    FFB_ROW(4, 8, 32, 1);
    FFB_ROW(4, 4, kThreads, 1);
    FFB_ROW(4, 8, kThreads, 1);
  }
  return static_cast<int>(cudaErrorInvalidValue);
}
#undef FFB_ROW

constexpr int kLnBlocks = 148 * 2;  // blocks (rows of partial sums) of the backward pass at most

// blocks of a launch whose blocks take `per` rows at a time
int ln_blocks(int64_t rows, int64_t per) {
  const int64_t want = (rows + per - 1) / per;
  return static_cast<int>(want < kLnBlocks ? want : kLnBlocks);
}
template <typename T>
int ln_bwd_blocks(int64_t rows, int c) {
  int blocks = 0;
  dispatch_row<T>(c, [&](auto, auto, auto g, auto u) {
    blocks = ln_blocks(rows, kThreads / decltype(g)::value * decltype(u)::value);
    return 0;
  });
  return blocks;
}

// A launch's shared memory: the teams' rings, three slots deep where they fit (two for fp32 rows of above
// 6000 channels with a residual), and room for the column sums behind them in time.
struct LnShared {
  int slots, bytes;
};
template <int V, int N, int G, int U>
LnShared ln_shared(std::initializer_list<int> row_bytes) {
  constexpr int team = G <= 32 ? 32 : kThreads, rows = team / G * U;
  int slot = 0;
  for (int b : row_bytes)
    if (b > 0) slot += slot_part(rows, b);
  slot *= kThreads / team;
  const int slots = kRing * slot <= 216 * 1024 ? kRing : 2;
  const int sums = G <= 32 ? kWarps * N * G * V * static_cast<int>(sizeof(float)) : 0;
  return {slots, slots * slot > sums ? slots * slot : sums};
}

template <typename T>
int ln_train(const LayerNormTrain& p, int* err, cudaStream_t stream) {
  return dispatch_row<T>(p.c, [&](auto v, auto n, auto g, auto u) {
    constexpr int V = decltype(v)::value, N = decltype(n)::value, G = decltype(g)::value, U = decltype(u)::value;
    const LnShared smem = ln_shared<V, N, G, U>({p.c * static_cast<int>(sizeof(T))});
    auto kernel = ln_train_kernel<T, V, N, G, U, kAnyRows>;
    if constexpr (V > 1) {
      if (p.c == V * N * G)
        kernel = ln_train_kernel<T, V, N, G, U, kFullRows>;
      else if (p.c % 16 == 0)
        kernel = ln_train_kernel<T, V, N, G, U, kWholeRows>;
    }
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem.bytes);
    if (e != cudaSuccess) return static_cast<int>(e);
    kernel<<<ln_blocks(p.rows, kThreads / G * U), kThreads, smem.bytes, stream>>>(
        static_cast<const T*>(p.x), static_cast<T*>(p.y), p.gamma, p.beta, p.mean, p.rstd, p.codes, p.scales, p.rows, p.c,
        p.eps, smem.slots, err);
    return static_cast<int>(cudaGetLastError());
  });
}

template <typename T>
int ln_bwd(const LayerNormBwd& p, int* err, cudaStream_t stream) {
  const bool mx = p.codes != nullptr;
  const int grid = ln_bwd_blocks<T>(p.rows, p.c);
  const bool sums = p.dgamma != nullptr || p.dbeta != nullptr;
  // one block writes the gradients itself; several leave rows [dgamma | dbeta] of partial sums
  float* part = static_cast<float*>(p.workspace);
  float* dg = !sums ? nullptr : grid == 1 ? p.dgamma : part;
  float* db = !sums ? nullptr : grid == 1 ? p.dbeta : part + p.c;
  const int row = p.c * static_cast<int>(sizeof(T));
  int rc = dispatch_row<T>(p.c, [&](auto v, auto n, auto g, auto u) {
    constexpr int V = decltype(v)::value, N = decltype(n)::value, G = decltype(g)::value, U = decltype(u)::value;
    const LnShared smem = ln_shared<V, N, G, U>({row, mx ? p.c : row, p.residual != nullptr ? row : 0});
    auto kernel = mx ? ln_bwd_kernel<T, V, N, G, U, true, kAnyRows> : ln_bwd_kernel<T, V, N, G, U, false, kAnyRows>;
    if constexpr (V > 1) {
      if (p.c == V * N * G)
        kernel = mx ? ln_bwd_kernel<T, V, N, G, U, true, kFullRows> : ln_bwd_kernel<T, V, N, G, U, false, kFullRows>;
      else if (p.c % 16 == 0)
        kernel = mx ? ln_bwd_kernel<T, V, N, G, U, true, kWholeRows> : ln_bwd_kernel<T, V, N, G, U, false, kWholeRows>;
    }
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem.bytes);
    if (e != cudaSuccess) return static_cast<int>(e);
    kernel<<<grid, kThreads, smem.bytes, stream>>>(
        static_cast<const T*>(p.dy), static_cast<const T*>(p.x), p.codes, p.scales, p.mean, p.rstd, p.gamma,
        static_cast<const T*>(p.residual), static_cast<T*>(p.dx), dg, db, 2 * static_cast<int64_t>(p.c), p.rows, p.c, smem.slots, err);
    return static_cast<int>(cudaGetLastError());
  });
  if (rc == 0 && sums && grid > 1) {
    rc = launch_after(ln_grad_reduce_kernel, (2 * p.c + 31) / 32, 1024, 0, stream, static_cast<const float*>(part), p.dgamma,
                      p.dbeta, grid, p.c);
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
  const int blocks = is_f32 ? ln_bwd_blocks<float>(rows, c) : ln_bwd_blocks<__nv_bfloat16>(rows, c);
  return blocks > 1 ? static_cast<size_t>(blocks) * 2 * c * sizeof(float) : 0;
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
