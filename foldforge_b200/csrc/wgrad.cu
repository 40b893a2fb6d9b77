// A linear layer's weight gradient dW [n, k] = dY^T X over `rows` rows, fp32 sums and output:
// dY [rows, n] bf16, X [rows, k] bf16 or its 8-bit checkpoint (mx8.cuh).
//
// The reduction runs along the rows, so both operands are MN-major for tcgen05: 64 rows of 64
// channels are one 128-byte-swizzled panel of 8 KB, exactly what a TMA box of a row-major tensor
// leaves in shared memory. Rows that TMA cannot take (widths that are not a multiple of 8 channels, a
// start off 16 bytes) are brought by the worker warps with aligned 16-byte loads and shifts. An 8-bit
// X is turned into bf16 on the way into shared memory (e4m3 times a power of two fits bf16's 8 bits of
// mantissa, so nothing is lost) and never exists in global memory. Loads run one or two stages ahead
// in registers.
//
// A pair tensor has rows = N^2 and n, k of a few hundred: few output tiles and a long reduction, so
// the rows are split over the SMs. A CTA takes one (128 MB) x BN tile of dW and one range of rows and
// leaves its fp32 sums in the workspace; wgrad_reduce_kernel adds the ranges in a fixed order.
//
// The tensor core truncates as it adds to a TMEM accumulator, and the bias grows with the number of
// additions (1.5e-6 of |dW| after 220 of them). So the products of kChunk stages go to one of two
// accumulators, and the worker warps add it to fp32 registers (round to nearest) while the other one
// fills: chains of 4 kChunk additions, however many rows there are.
#include <string.h>

#include <type_traits>

#include "abi_util.h"
#include "common.cuh"
#include "kernels.h"
#include "mx8.cuh"

namespace ffb {
namespace {

constexpr int kRows = 64;            // rows (the K of the product) of a stage
constexpr int kPanel = kRows * 128;  // bytes of a panel: 64 rows x 64 bf16 channels
constexpr int kWorkers = 16;         // warps that fill stages and drain accumulators
constexpr int kWorkerThreads = 32 * kWorkers;
constexpr int kWgradThreads = 64 + kWorkerThreads;
constexpr int kChunk = 8;            // stages of one accumulator
constexpr int kSms = 148;            // fixed, so that a result does not depend on the device's SM count

struct WgradParams {
  const __nv_bfloat16* dy;
  const __nv_bfloat16* x;
  const uint8_t* codes;
  const uint8_t* scales;
  float* out;          // dW, or the workspace of partial sums
  int64_t rows;
  int64_t split_rows;  // rows of a split, a multiple of kRows
  int n, k;
  int partial;         // leave partial sums instead of dW
  int* err;
};

template <int MB, int BN>
struct WgradSmem {
  static constexpr int kStageBytes = (2 * MB + BN / 64) * kPanel;
  static constexpr int kFit = (232448 - 2048) / kStageBytes;
  static constexpr int kStages = kFit < 6 ? kFit : 6;
  alignas(1024) uint8_t a[kStages][2 * MB * kPanel];
  alignas(1024) uint8_t b[kStages][BN / 64 * kPanel];
  uint64_t full[kStages];
  uint64_t empty[kStages];
  uint64_t acc_full[2];
  uint64_t acc_empty[2];
  uint32_t tmem_base;
};

// Both operands MN-major, bf16 -> fp32.
__host__ __device__ constexpr uint32_t idesc_bf16_f32_abmn(int m, int n) {
  return idesc_bf16_f32(m, n) | (1u << 15) | (1u << 16);
}

enum Operand : int {
  kByTma,         // bf16 rows of a multiple of 8 channels, 16-byte aligned
  kByWorkers,     // bf16 rows of any width and alignment
  kCodes,         // a checkpoint with rows of a multiple of 8 codes, 8-byte aligned
  kCodesAnyhow,   // a checkpoint of any width and alignment
};

// A worker thread's share of one operand: 8 channels (a 16-byte piece of a panel) of PANELS rows of each
// stage, kStep rows apart. Eight threads lie along a panel's row, then come the panels, then the rows.
// `load` issues a stage's loads, `store` writes its panels; `raw` holds what is in between.
//
// Rows of any width: the 16 bytes of 8 bf16 channels start at any even address. Two aligned 16-byte
// loads cover them, and a shift that is the same for all of a thread's pieces (kStep rows are a multiple
// of 16 bytes whatever the width) picks them out; for codes, 8 bytes by two 8-byte loads. What lies past
// the row's end is the next row's and reaches only columns of dW that are not written. An aligned load
// that would leave the tensor is put together from the elements inside it.
template <Operand KIND, int PANELS>
struct Share {
  static constexpr bool kIsCodes = KIND == kCodes || KIND == kCodesAnyhow;
  static constexpr int kStep = kRows / PANELS;
  static constexpr int kBytes = kIsCodes ? 8 : 16;  // of a piece in memory
  using Word = std::conditional_t<kIsCodes, uint2, uint4>;
  struct Raw {
    Word lo, hi;  // hi: not for kCodes
    uint32_t scale;
  };
  const uint8_t* at;     // the piece of the first row of the next stage to load
  const uint8_t* scale;  // the scale of that piece
  const uint8_t *begin, *end;  // of the tensor
  int64_t stride;        // bytes of a row
  int blocks;            // scales of a row
  int64_t left;          // rows of the split from the thread's first row of the next stage on; none if the channels lie past the row
  uint32_t offset;       // of the first piece in the stage's panels
  uint32_t shift;        // bytes from the aligned load's start to the piece

  __device__ __forceinline__ Share(const void* base, const uint8_t* scales, int64_t rows, int width, int col0, int64_t first,
                                   int64_t last, int id) {
    const int chunk = id & 7, panel = (id >> 3) % PANELS, row = id / (8 * PANELS);
    const int col = col0 + panel * 64 + chunk * 8;
    constexpr int size = kIsCodes ? 1 : 2;
    begin = static_cast<const uint8_t*>(base);
    end = begin + rows * width * size;
    stride = static_cast<int64_t>(width) * size;
    at = begin + (first + row) * stride + static_cast<int64_t>(col) * size;
    blocks = (width + kMxBlock - 1) / kMxBlock;
    scale = kIsCodes ? scales + (first + row) * blocks + col / kMxBlock : nullptr;
    left = col < width ? last - first - row : 0;
    offset = panel * kPanel + sw128_offset(row, chunk * 8);
    shift = KIND == kCodes ? 0 : static_cast<uint32_t>(reinterpret_cast<uintptr_t>(at) & (kBytes - 1));
  }

  __device__ __forceinline__ void load(Raw (&raw)[PANELS]) {
#pragma unroll
    for (int i = 0; i < PANELS; ++i) {
      Raw& r = raw[i];
      r.lo = r.hi = Word{};
      r.scale = 0;
      if (i * kStep < left) {
        const uint8_t* q = at + i * kStep * stride - shift;
        if constexpr (kIsCodes) r.scale = __ldg(scale + static_cast<int64_t>(i * kStep) * blocks);
        if constexpr (KIND == kCodes) {
          r.lo = __ldg(reinterpret_cast<const Word*>(q));
        } else if (q >= begin && q + 2 * kBytes <= end) {
          r.lo = __ldg(reinterpret_cast<const Word*>(q));
          r.hi = __ldg(reinterpret_cast<const Word*>(q + kBytes));
        } else {
          r.lo = edge(q);
          r.hi = edge(q + kBytes);
        }
      }
    }
    at += kRows * stride;
    if (kIsCodes) scale += kRows * static_cast<int64_t>(blocks);
    left -= kRows;
  }

  // the aligned bytes at q, 0 where they lie outside the tensor (elements start at even addresses)
  __device__ __noinline__ Word edge(const uint8_t* q) const {
    constexpr int size = kIsCodes ? 1 : 2;
    uint32_t w[kBytes / 4] = {};
#pragma unroll
    for (int i = 0; i < kBytes; i += size)
      if (q + i >= begin && q + i < end)
        w[i / 4] |= (kIsCodes ? static_cast<uint32_t>(__ldg(q + i)) : static_cast<uint32_t>(__ldg(reinterpret_cast<const uint16_t*>(q + i))))
                    << (8 * (i & 3));
    if constexpr (kIsCodes)
      return make_uint2(w[0], w[1]);
    else
      return make_uint4(w[0], w[1], w[2], w[3]);
  }

  __device__ __forceinline__ uint4 value(const Raw& r) const {
    if constexpr (kIsCodes) {
      uint2 c = r.lo;
      if constexpr (KIND == kCodesAnyhow) {
        const uint32_t bits = (shift & 3u) * 8;
        const uint32_t w0 = shift & 4u ? r.lo.y : r.lo.x, w1 = shift & 4u ? r.hi.x : r.lo.y;
        const uint32_t w2 = shift & 4u ? r.hi.y : r.hi.x;
        c = make_uint2(__funnelshift_r(w0, w1, bits), __funnelshift_r(w1, w2, bits));
      }
      float f[8];
      mx_decode<8>(c, mx_scale(r.scale), f);
      return make_uint4(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]), pack_bf16(f[4], f[5]), pack_bf16(f[6], f[7]));
    } else {
      uint32_t w[8] = {r.lo.x, r.lo.y, r.lo.z, r.lo.w, r.hi.x, r.hi.y, r.hi.z, r.hi.w};
#pragma unroll
      for (int i = 0; i < 6; ++i) w[i] = shift & 8u ? w[i + 2] : w[i];
#pragma unroll
      for (int i = 0; i < 5; ++i) w[i] = shift & 4u ? w[i + 1] : w[i];
      const uint32_t bits = (shift & 2u) * 8;
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], bits);
      return make_uint4(w[0], w[1], w[2], w[3]);
    }
  }

  __device__ __forceinline__ void store(uint8_t* panels, const Raw (&raw)[PANELS]) const {
#pragma unroll
    for (int i = 0; i < PANELS; ++i) *reinterpret_cast<uint4*>(panels + offset + i * kStep * 128) = value(raw[i]);
  }
};

template <int PANELS>
struct Share<kByTma, PANELS> {
  struct Raw {};
  __device__ __forceinline__ Share(const void*, const uint8_t*, int64_t, int, int, int64_t, int64_t, int) {}
  __device__ __forceinline__ void load(Raw (&)[PANELS]) {}
  __device__ __forceinline__ void store(uint8_t*, const Raw (&)[PANELS]) const {}
};

template <int MB, int BN, Operand A, Operand B>
__global__ void __launch_bounds__(kWgradThreads, 1)
    wgrad_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, WgradParams p) {
  using Smem = WgradSmem<MB, BN>;
  constexpr int kStages = Smem::kStages;
  constexpr int kColumns = MB * BN;            // TMEM columns of an accumulator: 64, 128 or 256
  constexpr int kMine = kColumns / (kWorkers / 4);  // columns a worker warp drains (of its 32 lanes)
  constexpr bool kTma = A == kByTma || B == kByTma, kFill = A != kByTma || B != kByTma;
  static_assert(kStages < kChunk, "a chunk is drained kStages stages after its end");
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  Smem& s = *reinterpret_cast<Smem*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int tiles_k = (p.k + BN - 1) / BN;
  const int tile_n = blockIdx.x / tiles_k, tile_k = blockIdx.x - tile_n * tiles_k;
  const int n0 = tile_n * 128 * MB, k0 = tile_k * BN;
  const int64_t first = static_cast<int64_t>(blockIdx.y) * p.split_rows;
  const int64_t end = first + p.split_rows < p.rows ? first + p.split_rows : p.rows;
  const int steps = static_cast<int>((end - first + kRows - 1) / kRows);

  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&s.full[i], (kTma ? 1 : 0) + (kFill ? kWorkers : 0));
      mbar_init(&s.empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s.acc_full[i], 1);
      mbar_init(&s.acc_empty[i], kWorkers);
    }
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(&s.tmem_base, 2 * kColumns);
    tmem_relinquish();
  }
  if (warp == 0 && lane == 0) {
    if (A == kByTma) tma_prefetch_map(&map_a);
    if (B == kByTma) tma_prefetch_map(&map_b);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s.tmem_base;

  if (warp == 0) {
    if (kTma && lane == 0) {
      int it = 0;
      for (; it < steps; ++it) {
        const int st = it % kStages;
        if (!mbar_wait(&s.empty[st], ((it / kStages) & 1) ^ 1, p.err, kErrTimeoutEmpty)) break;
        const int row = static_cast<int>(first + static_cast<int64_t>(it) * kRows);
        // panels wholly past the matrix are not loaded (their part of dW is not written)
        int bytes = 0;
        if (A == kByTma)
          for (int q = 0; q < 2 * MB; ++q) bytes += n0 + 64 * q < p.n ? kPanel : 0;
        if (B == kByTma)
          for (int q = 0; q < BN / 64; ++q) bytes += k0 + 64 * q < p.k ? kPanel : 0;
        mbar_arrive_expect_tx(&s.full[st], bytes);
        if (A == kByTma)
          for (int q = 0; q < 2 * MB; ++q)
            if (n0 + 64 * q < p.n) tma_load_2d(s.a[st] + q * kPanel, &map_a, &s.full[st], n0 + 64 * q, row);
        if (B == kByTma)
          for (int q = 0; q < BN / 64; ++q)
            if (k0 + 64 * q < p.k) tma_load_2d(s.b[st] + q * kPanel, &map_b, &s.full[st], k0 + 64 * q, row);
      }
      // every issued stage must land before the CTA may exit
      for (int j = it > kStages ? it - kStages : 0; j < it; ++j)
        mbar_wait(&s.full[j % kStages], (j / kStages) & 1, p.err, kErrTimeoutLoad);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t idesc = idesc_bf16_f32_abmn(128, BN);
      for (int it = 0; it < steps; ++it) {
        const int st = it % kStages, chunk = it / kChunk;
        if (it % kChunk == 0 &&
            !mbar_wait(&s.acc_empty[chunk & 1], ((chunk >> 1) & 1) ^ 1, p.err, kErrTimeoutEmpty))
          break;
        if (!mbar_wait(&s.full[st], (it / kStages) & 1, p.err, kErrTimeoutLoad)) break;
        tc_fence_after();
        const uint32_t a = smem_u32(s.a[st]), b = smem_u32(s.b[st]);
        const uint32_t d = tmem + (chunk & 1) * kColumns;
#pragma unroll
        for (int kk = 0; kk < kRows / 16; ++kk) {
          // 16 rows further: two 8-row groups of 1024 bytes
          const uint64_t db = desc_mnmajor_sw128(b + kk * 2048, kPanel, 1024);
#pragma unroll
          for (int m = 0; m < MB; ++m)
            mma_bf16(d + m * BN, desc_mnmajor_sw128(a + m * 2 * kPanel + kk * 2048, kPanel, 1024), db, idesc,
                     (it % kChunk | kk) != 0);
        }
        mma_commit(&s.empty[st]);
        if (it % kChunk == kChunk - 1 || it == steps - 1) mma_commit(&s.acc_full[chunk & 1]);
      }
    }
  } else {
    const int id = threadIdx.x - 64;
    const int quarter = warp & 3, group = (warp - 2) / 4;  // TMEM lanes 32 quarter.., columns kMine group..
    const uint32_t mine = (static_cast<uint32_t>(quarter * 32) << 16) + group * kMine;
    float acc[kMine];
#pragma unroll
    for (int i = 0; i < kMine; ++i) acc[i] = 0.f;
    int drained = 0;
    bool ok = true;
    auto drain = [&]() {
      const int set = drained & 1;
      ok = mbar_wait(&s.acc_full[set], (drained >> 1) & 1, p.err, kErrTimeoutMma);
      ok = __all_sync(0xFFFFFFFFu, ok);
      if (!ok) return;
      tc_fence_after();
      const uint32_t at = tmem + set * kColumns + mine;
#pragma unroll
      for (int c = 0; c < kMine; c += 16) {  // 16 columns at a time: the sums leave few registers
        uint32_t v[16];
        tmem_ld16(at + c, v);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[c + i] += __uint_as_float(v[i]);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&s.acc_empty[set]);
      ++drained;
    };
    if constexpr (kFill) {
      // loads run kAhead stages ahead of the stage being written
      constexpr int kAhead = A == kByTma && B == kCodes && BN <= 128 ? 2 : 1;  // as the registers allow
      using ShareA = Share<A, 2 * MB>;
      using ShareB = Share<B, BN / 64>;
      ShareA sa(p.dy, nullptr, p.rows, p.n, n0, first, end, id);
      ShareB sb(p.codes != nullptr ? static_cast<const void*>(p.codes) : p.x, p.scales, p.rows, p.k, k0, first, end, id);
      typename ShareA::Raw ra[kAhead][2 * MB];
      typename ShareB::Raw rb[kAhead][BN / 64];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        sa.load(ra[u]);
        sb.load(rb[u]);
      }
      for (int base = 0; base < steps && ok; base += kAhead) {
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          const int it = base + u;
          if (it < steps && ok) {
            const int st = it % kStages;
            ok = mbar_wait(&s.empty[st], ((it / kStages) & 1) ^ 1, p.err, kErrTimeoutEmpty);
            ok = __all_sync(0xFFFFFFFFu, ok);
            if (ok) {
              sa.store(s.a[st], ra[u]);
              sb.store(s.b[st], rb[u]);
              fence_async_smem();
              __syncwarp();
              if (lane == 0) mbar_arrive(&s.full[st]);
              sa.load(ra[u]);  // nothing past the split's rows
              sb.load(rb[u]);
              // this stage was free because the MMAs up to kStages stages ago are complete, the chunk
              // before this one's among them
              if (it >= kChunk && it % kChunk == kStages) drain();
            }
          }
        }
      }
    }
    for (const int chunks = (steps + kChunk - 1) / kChunk; ok && drained < chunks;) drain();
    if (ok) {
      const int nn = n0 + (group * kMine / BN) * 128 + quarter * 32 + lane;
      const int kk = k0 + group * kMine % BN;
      if (p.partial) {
        // [split][tile][column / 4][128 MB rows][4]: a warp writes 512 bytes in one piece
        float4* o = reinterpret_cast<float4*>(p.out) +
                    (static_cast<int64_t>(blockIdx.y) * gridDim.x + blockIdx.x) * (128 * MB * BN / 4) + (nn - n0) +
                    (group * kMine % BN / 4) * (128 * MB);
        if (nn < p.n) {
#pragma unroll
          for (int i = 0; i < kMine / 4; ++i)
            if (kk + 4 * i < p.k) o[i * (128 * MB)] = make_float4(acc[4 * i], acc[4 * i + 1], acc[4 * i + 2], acc[4 * i + 3]);
        }
      } else if (nn < p.n) {
        float* o = p.out + static_cast<int64_t>(nn) * p.k + kk;
        if ((reinterpret_cast<uintptr_t>(p.out) & 15u) == 0 && p.k % 4 == 0) {
#pragma unroll
          for (int i = 0; i < kMine / 4; ++i)
            if (kk + 4 * i < p.k)
              reinterpret_cast<float4*>(o)[i] = make_float4(acc[4 * i], acc[4 * i + 1], acc[4 * i + 2], acc[4 * i + 3]);
        } else {
#pragma unroll
          for (int i = 0; i < kMine; ++i)
            if (kk + i < p.k) o[i] = acc[i];
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, 2 * kColumns);
  }
}

// dW = the splits' partial sums, added in a fixed order: a thread takes four channels of a row of dW and
// every eighth split, then the eight sums of a place are added in turn.
__global__ void __launch_bounds__(256)
    wgrad_reduce_kernel(const float4* __restrict__ part, float* __restrict__ out, int splits, int n, int k, int tile_rows,
                        int bn, int tiles_k, int64_t tile_stride, int64_t split_stride) {
  __shared__ float4 sum[8][32];
  const int lane = threadIdx.x & 31, g = threadIdx.x / 32;
  const int row_blocks = (n + 31) / 32;
  const int rb = blockIdx.x % row_blocks, c4 = blockIdx.x / row_blocks;  // 32 rows of one column of four channels
  const int row = rb * 32 + lane, col = c4 * 4;
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
  if (row < n) {
    const int tn = row / tile_rows, tk = col / bn;
    const float4* p = part + (static_cast<int64_t>(tn) * tiles_k + tk) * tile_stride + (row - tn * tile_rows) +
                      static_cast<int64_t>(col - tk * bn) / 4 * tile_rows;
#pragma unroll 4
    for (int s = g; s < splits; s += 8) {
      const float4 v = p[s * split_stride];
      a.x += v.x;
      a.y += v.y;
      a.z += v.z;
      a.w += v.w;
    }
  }
  sum[g][lane] = a;
  __syncthreads();
  if (g == 0 && row < n) {
#pragma unroll
    for (int i = 1; i < 8; ++i) {
      const float4 v = sum[i][lane];
      a.x += v.x;
      a.y += v.y;
      a.z += v.z;
      a.w += v.w;
    }
    float* o = out + static_cast<int64_t>(row) * k + col;
    const float w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (col + i < k) o[i] = w[i];
  }
}

struct WgradPlan {
  int mb, bn, tiles, tiles_k, splits;
  int64_t split_rows;
  size_t workspace() const { return splits > 1 ? static_cast<size_t>(splits) * tiles * 128 * mb * bn * sizeof(float) : 0; }
};

// `workers`: an operand comes by shifted loads, which take the worker warps' registers: tiles of 128 x 128
// at most. Otherwise 256 x 128, or 128 x 256 for few dY channels: larger tiles read each
// operand less often.
WgradPlan plan(int64_t rows, int n, int k, bool workers) {
  WgradPlan p;
  p.mb = n <= 128 || workers ? 1 : 2;
  p.bn = k <= 64 ? 64 : p.mb == 1 && !workers && k > 128 && (k - 1) % 256 >= 128 ? 256 : 128;
  p.tiles_k = (k + p.bn - 1) / p.bn;
  const int64_t tiles = static_cast<int64_t>((n + 128 * p.mb - 1) / (128 * p.mb)) * p.tiles_k;
  p.tiles = static_cast<int>(tiles);
  // The number of splits that ends first, in stages: waves of CTAs, each with its own start and end (about
  // 6 stages' time), and for the partial sums a second kernel and a pass over them.
  const int64_t steps = (rows + kRows - 1) / kRows;
  int64_t best = 1, best_cost = -1;
  for (int64_t s = 1; s <= kSms && s <= steps; ++s) {
    if (s > 1 && tiles * s > 4 * kSms) break;  // enough tiles to fill the SMs
    const int64_t waves = (tiles * s + kSms - 1) / kSms;
    const int64_t cost = waves * ((steps + s - 1) / s + 6) + (s > 1 ? 6 + s / 16 : 0);
    if (best_cost < 0 || cost < best_cost) {
      best = s;
      best_cost = cost;
    }
  }
  const int64_t per = (steps + best - 1) / best;
  p.split_rows = per * kRows;
  p.splits = static_cast<int>((steps + per - 1) / per);  // no empty split
  return p;
}

template <int MB, int BN, Operand A, Operand B>
int launch(const CUtensorMap& a, const CUtensorMap& b, const WgradParams& p, const WgradPlan& plan, cudaStream_t stream) {
  constexpr size_t smem = sizeof(WgradSmem<MB, BN>) + 1024;
  static_assert(smem <= 232448, "weight-gradient shared memory exceeds the per-CTA limit");
  auto kernel = wgrad_kernel<MB, BN, A, B>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
  if (e != cudaSuccess) return static_cast<int>(e);
  kernel<<<dim3(plan.tiles, plan.splits), kWgradThreads, smem, stream>>>(a, b, p);
  return static_cast<int>(cudaGetLastError());
}

// tiles of 128 x 64 and 128 x 128, for operands by shifted loads
template <Operand A, Operand B>
int launch_small(const CUtensorMap& a, const CUtensorMap& b, const WgradParams& p, const WgradPlan& plan, cudaStream_t s) {
  return plan.bn == 64 ? launch<1, 64, A, B>(a, b, p, plan, s) : launch<1, 128, A, B>(a, b, p, plan, s);
}

// every tile, for operands that leave the workers' registers alone
template <Operand A, Operand B>
int launch_any(const CUtensorMap& a, const CUtensorMap& b, const WgradParams& p, const WgradPlan& plan, cudaStream_t s) {
  if (plan.mb == 2) return plan.bn == 64 ? launch<2, 64, A, B>(a, b, p, plan, s) : launch<2, 128, A, B>(a, b, p, plan, s);
  return plan.bn == 256 ? launch<1, 256, A, B>(a, b, p, plan, s) : launch_small<A, B>(a, b, p, plan, s);
}

int panel_map(CUtensorMap* map, const void* base, int64_t rows, int width) {
  const uint64_t dims[2] = {static_cast<uint64_t>(width), static_cast<uint64_t>(rows)};
  const uint64_t strides[1] = {static_cast<uint64_t>(width) * 2};
  const uint32_t box[2] = {64, kRows};
  return make_map(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, base, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

bool by_tma(const void* base, int width) { return (reinterpret_cast<uintptr_t>(base) & 15u) == 0 && width % 8 == 0; }

}  // namespace

size_t weight_grad_workspace_bytes(int64_t rows, int n, int k) {
  // the tensors' alignment is not known here: room for either plan
  const size_t a = plan(rows, n, k, false).workspace(), b = plan(rows, n, k, true).workspace();
  return a > b ? a : b;
}

int weight_grad_forward(const void* dy, const void* x, const uint8_t* codes, const uint8_t* scales, float* dw,
                        void* workspace, int64_t rows, int n, int k, const DeviceInfo& info, cudaStream_t stream) {
  const bool a_tma = by_tma(dy, n), b_tma = codes == nullptr && by_tma(x, k);
  const bool whole = codes != nullptr && (reinterpret_cast<uintptr_t>(codes) & 7u) == 0 && k % 8 == 0;
  const WgradPlan pl = plan(rows, n, k, !a_tma || !(b_tma || whole));
  CUtensorMap ma, mb;
  memset(&ma, 0, sizeof(ma));
  memset(&mb, 0, sizeof(mb));
  int st = a_tma ? panel_map(&ma, dy, rows, n) : 0;
  if (st == 0 && b_tma) st = panel_map(&mb, x, rows, k);
  if (st != 0) return st;
  WgradParams p;
  p.dy = static_cast<const __nv_bfloat16*>(dy);
  p.x = static_cast<const __nv_bfloat16*>(x);
  p.codes = codes;
  p.scales = scales;
  p.rows = rows;
  p.split_rows = pl.split_rows;
  p.n = n;
  p.k = k;
  p.partial = pl.splits > 1;
  p.out = p.partial ? static_cast<float*>(workspace) : dw;
  p.err = info.err;
  int rc;
  if (a_tma)
    rc = b_tma ? launch_any<kByTma, kByTma>(ma, mb, p, pl, stream)
         : whole ? launch_any<kByTma, kCodes>(ma, mb, p, pl, stream)
         : codes ? launch_small<kByTma, kCodesAnyhow>(ma, mb, p, pl, stream)
                 : launch_small<kByTma, kByWorkers>(ma, mb, p, pl, stream);
  else
    rc = b_tma ? launch_small<kByWorkers, kByTma>(ma, mb, p, pl, stream)
         : whole ? launch_small<kByWorkers, kCodes>(ma, mb, p, pl, stream)
         : codes ? launch_small<kByWorkers, kCodesAnyhow>(ma, mb, p, pl, stream)
                 : launch_small<kByWorkers, kByWorkers>(ma, mb, p, pl, stream);
  if (rc == 0 && p.partial) {
    const int rows_of_tile = 128 * pl.mb;
    const int64_t tile_stride = static_cast<int64_t>(rows_of_tile) * pl.bn / 4;
    wgrad_reduce_kernel<<<((n + 31) / 32) * ((k + 3) / 4), 256, 0, stream>>>(
        static_cast<const float4*>(workspace), dw, pl.splits, n, k, rows_of_tile, pl.bn, pl.tiles_k, tile_stride,
        tile_stride * pl.tiles);
    rc = static_cast<int>(cudaGetLastError());
  }
  return cuda_status(rc, "weight_grad launch");
}

}  // namespace ffb
