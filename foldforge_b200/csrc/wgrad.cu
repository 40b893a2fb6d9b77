// A linear layer's weight gradient dW [n, k] = dY^T X over `rows` rows, fp32 sums and output:
// dY [rows, n] bf16, X [rows, k] bf16 or its 8-bit checkpoint (mx8.cuh).
//
// The reduction runs along the rows, so both operands are MN-major for tcgen05: 64 rows of 64
// channels are one 128-byte-swizzled panel of 8 KB, exactly what a TMA box of a row-major tensor
// leaves in shared memory. An 8-bit X is turned into bf16 on the way into the panels (e4m3 times a
// power of two fits bf16's 8 bits of mantissa, so nothing is lost) and never exists in global memory.
// Rows that neither way takes (widths that are not a multiple of 8 channels of bf16 or 16 codes) are first
// copied into the workspace as bf16 with rows of a multiple of 8.
//
// X is the M side and dY the N side: a product of 128 x 256 x 16 reads 12 KB of shared memory in its 128
// cycles, two of 128 x 128 read 16 KB and run at 0.7 of the rate; and a warp's store of sums, 32 lanes of M,
// is 32 neighbours of a row of dW.
//
// A pair tensor has rows = N^2 and n, k of a few hundred: few output tiles and a long reduction, so
// the rows are split over the SMs. A CTA takes one BN x (128 MB) tile of dW and one range of rows and
// leaves its fp32 sums in the workspace; wgrad_reduce_kernel adds the ranges in a fixed order.
//
// The tensor core truncates as it adds to a TMEM accumulator, and the bias grows with the number of
// additions (1.5e-6 of |dW| after 220 of them). So the products of kChunk stages go to one of two
// accumulators, and the warps add it to fp32 registers (round to nearest) while the other one
// fills: chains of 4 kChunk additions, however many rows there are (2e-7 of |dW|).
//
// Measured on one B200: n 512, k 128, 262144 rows with an 8-bit X (303 MB, 34 GFLOP; 46 us of copying, 21 us
// of tensor work) in 52 us + 4 us for the sum over the splits. It waits for memory:
// with 128 KB of dY in flight an SM, 5.8 TB/s means a latency of about 3 us (by count, not measured). Steps on
// the way, each timed with the L2 full of lines to write back: loads and conversions in turn 156 us, a stage
// ahead in registers 90, codes by cp.async and the warps in groups 70, 256 channels of dY as the N side 65 to
// 68; the same kernel that took 68 so took 52 over clean lines, the way all times here are taken. In a loop
// over three inputs 64 us with the sum; 3 groups of fill warps 64, chunks of 16 stages 65.
// Rows that have to be padded (n 129, k 68, 90000 rows): 14 us for that, 12 for the products, 4 for the sum.
// Reading such rows through the codes' rings took 97 us for the products alone (lines to write back) where
// padding and products took 18 + 14.
// A bf16 library product with a bf16 result takes 60.3 us for the first of these (65 to 66 here, from bf16 or 8 bits),
// 10.9 for 512 rows of 1536 and 384 (10.4 from bf16, 12.4 from 8 bits) and 251 for the odd widths (29).
#include <string.h>

#include "abi_util.h"
#include "common.cuh"
#include "kernels.h"
#include "launch.cuh"
#include "mx8.cuh"

namespace ffb {
namespace {

constexpr int kRows = 64;            // rows (the K of the product) of a stage
constexpr int kPanel = kRows * 128;  // bytes of a panel: 64 rows x 64 bf16 channels
constexpr int kWarps = 16;           // 0: TMA, 1: products, the last ones: an 8-bit X; all of them drain accumulators
constexpr int kWgradThreads = 32 * kWarps;
constexpr int kChunk = 8;            // stages of one accumulator
constexpr int kSms = 148;            // fixed, so that a result does not depend on the device's SM count
constexpr int kSmem = 232448 - 2048;  // shared memory of a CTA, less alignment and barriers

struct WgradParams {
  const uint8_t* codes;  // X's checkpoint, null where X comes by TMA
  const uint8_t* scales;
  float* out;            // dW, or a dW of partial sums for each split
  int64_t rows;
  int64_t split_rows;    // rows of a split, a multiple of kRows
  int n, k;
  int* err;
};

// Both operands MN-major, bf16 -> fp32.
__host__ __device__ constexpr uint32_t idesc_bf16_f32_abmn(int m, int n) {
  return idesc_bf16_f32(m, n) | (1u << 15) | (1u << 16);
}

// ---- an 8-bit X. The fill warps work in kGroups groups of four, each on every kGroups'th stage, so that one
// group's waits and fences lie beside the other's work. A warp takes 16 consecutive rows of its group's
// stage: it copies their codes and scales as they lie in memory to its own part of a ring in shared memory
// (cp.async, kSlots of its stages ahead), and later turns them into panels. Nothing but the finished
// panels is shared between warps.
constexpr int kGroups = 2;
constexpr int kSlots = 2;
constexpr int kFillStages = 3;
constexpr int kWarpRows = kRows / 4;

__device__ __forceinline__ void copy_async_16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy_async_4(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT>
__device__ __forceinline__ void copy_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory");
}

// The aligned word at q of a byte tensor [begin, end); 0 for bytes outside it, which are never read, and
// for all of them without `in`.
__device__ __forceinline__ void copy_word(uint32_t dst, const uint8_t* q, bool in, const uint8_t* begin, const uint8_t* end) {
  if (in && q < begin) {
    for (int i = 0; i < 4; ++i) {
      const uint32_t byte = q + i >= begin && q + i < end ? __ldg(q + i) : 0;
      asm volatile("st.shared.u8 [%0], %1;" ::"r"(dst + i), "r"(byte) : "memory");
    }
    return;
  }
  const int bytes = !in ? 0 : end - q < 4 ? static_cast<int>(end - q) : 4;
  // with no bytes to copy nothing is read; the address is a valid one all the same
  copy_async_4(dst, in ? q : begin - (reinterpret_cast<uintptr_t>(begin) & 3u), bytes);
}

// A fill warp's rows of codes (a multiple of 16 of them, 16-byte aligned); its scales at any address: a row
// takes the aligned words that cover them.
template <int PANELS>
struct CodeRows {
  static constexpr int kSpan = PANELS * 64;                // bytes of a row that the tile wants
  static constexpr int kGranules = kSpan / 16;
  static constexpr int kRowsAtOnce = 32 / kGranules;       // rows that one instruction copies
  static constexpr int kScaleWords = PANELS == 4 ? 3 : 2;  // 4-byte words that cover the row's scales
  static constexpr int kPitch = kSpan + 16;                // of a row in the ring, scales behind the codes
  static constexpr int kSlot = kWarpRows * kPitch;

  const uint8_t* from;        // this lane's 16 codes of the first row(s) of the warp's next stage to copy
  const uint8_t* from_scale;  // the first scale of the warp's first row there
  int left;                   // rows of the split from the warp's first row there
  int lane, row;              // the warp's first row in a stage

  __device__ __forceinline__ static int blocks(int k) { return (k + kMxBlock - 1) / kMxBlock; }

  __device__ __forceinline__ CodeRows(const WgradParams& p, int k0, int64_t first, int64_t end, int row_in_split, int lane_)
      : lane(lane_), row(row_in_split % kRows) {
    first += row_in_split;
    left = static_cast<int>(end - first);
    from = p.codes + (first + lane / kGranules) * p.k + k0 + lane % kGranules * 16;
    from_scale = p.scales + first * blocks(p.k) + k0 / kMxBlock;
  }

  // the warp's rows of its next stage; rows past the split's end and codes past the row's become 0
  __device__ __forceinline__ void copy(uint32_t ring, const WgradParams& p, int k0) {
    const int j0 = lane / kGranules, i0 = lane % kGranules;
#pragma unroll
    for (int j = 0; j < kWarpRows; j += kRowsAtOnce) {
      const bool in = j + j0 < left && k0 + 16 * i0 < p.k;
      copy_async_16(ring + (j + j0) * kPitch + i0 * 16, in ? from + static_cast<int64_t>(j) * p.k : p.codes, in ? 16 : 0);
    }
    from += static_cast<int64_t>(kGroups * kRows) * p.k;
    const int n = blocks(p.k);
    const uint32_t low = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(from_scale));
#pragma unroll
    for (int g = 0; g < kWarpRows * kScaleWords; g += 32) {
      const int at = g + lane, j = at / kScaleWords, i = at - j * kScaleWords;
      if (kWarpRows * kScaleWords % 32 == 0 || at < kWarpRows * kScaleWords) {
        const int shift = static_cast<int>((low + j * n) & 3u);
        const int count = n - k0 / kMxBlock < kSpan / kMxBlock ? n - k0 / kMxBlock : kSpan / kMxBlock;
        copy_word(ring + j * kPitch + kSpan + i * 4, from_scale + static_cast<int64_t>(j) * n - shift + 4 * i,
                  j < left && 4 * i < shift + count, p.scales, p.scales + p.rows * n);
      }
    }
    from_scale += static_cast<int64_t>(kGroups * kRows) * n;
    left -= kGroups * kRows;
  }

  // The warp's rows from the ring to a stage's panels: eight lanes along a panel's row, then the panels,
  // then the rows. Four pieces at a time are read before the first is written: the compiler cannot know
  // that panels and ring are apart, and one piece after the other would wait out each read.
  __device__ __forceinline__ void fill(uint8_t* panels, const uint8_t* ring, const WgradParams& p) const {
    constexpr int kRowLanes = 8 * PANELS;
    const uint32_t low = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(from_scale));  // 64 rows later: the same low bits
    const int n = blocks(p.k);
#pragma unroll
    for (int first = 0; first < PANELS * kWarpRows / 4; first += 4) {
      uint2 c[4];
      uint32_t scale[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int at = (first + i) * 32 + lane, j = at / kRowLanes, chunk = at % kRowLanes;
        c[i] = *reinterpret_cast<const uint2*>(ring + j * kPitch + 8 * chunk);
        scale[i] = ring[j * kPitch + kSpan + ((low + j * n) & 3u) + chunk / 4];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int at = (first + i) * 32 + lane, j = at / kRowLanes, chunk = at % kRowLanes;
        *reinterpret_cast<uint4*>(panels + (chunk / 8) * kPanel + sw128_offset(row + j, (chunk & 7) * 8)) =
            mx_decode_bf16(c[i], scale[i]);
      }
    }
  }
};

// The ring that TMA fills holds dY's panels and, unless CODES, X's behind them; an 8-bit X has a ring of its
// own, so that dY's loads can run further ahead.
template <int MB, int BN, bool CODES>
struct WgradSmem {
  static constexpr int kTmaPanels = BN / 64 + (CODES ? 0 : 2 * MB);
  static constexpr int kFillBytes = CODES ? kFillStages * 2 * MB * kPanel : 0;
  static constexpr int kRing = CODES ? kSlots * CodeRows<2 * MB>::kSlot : 0;  // of a fill warp
  static constexpr int kFit = (kSmem - kFillBytes - 4 * kGroups * kRing) / (kTmaPanels * kPanel);
  static constexpr int kStages = kFit < 6 ? kFit : 6;
  alignas(1024) uint8_t tma[kStages][kTmaPanels * kPanel];
  alignas(1024) uint8_t fill[kFillBytes + 1024];
  alignas(16) uint8_t ring[4 * kGroups][kRing + 16];
  uint64_t full[kStages];
  uint64_t empty[kStages];
  uint64_t fill_full[kFillStages];
  uint64_t fill_empty[kFillStages];
  uint64_t acc_full[2];
  uint64_t acc_empty[2];
  uint32_t tmem_base;
};

template <int MB, int BN, bool CODES>
__global__ void __launch_bounds__(kWgradThreads, 1)
    wgrad_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_dy, WgradParams p) {
  using Smem = WgradSmem<MB, BN, CODES>;
  constexpr int kStages = Smem::kStages;
  constexpr int kColumns = MB * BN;                // TMEM columns of an accumulator: 64, 128 or 256
  constexpr int kMine = kColumns / (kWarps / 4);   // columns a warp drains (of its 32 lanes)
  static_assert(kStages >= 3 && kStages < kChunk, "stages");
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  Smem& s = *reinterpret_cast<Smem*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int tiles_k = (p.k + 128 * MB - 1) / (128 * MB);
  const int tile_n = blockIdx.x / tiles_k, tile_k = blockIdx.x - tile_n * tiles_k;
  const int n0 = tile_n * BN, k0 = tile_k * 128 * MB;
  const int64_t first = static_cast<int64_t>(blockIdx.y) * p.split_rows;
  const int64_t end = first + p.split_rows < p.rows ? first + p.split_rows : p.rows;
  const int steps = static_cast<int>((end - first + kRows - 1) / kRows);
  const int chunks = (steps + kChunk - 1) / kChunk;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&s.full[i], 1);
      mbar_init(&s.empty[i], 1);
    }
    for (int i = 0; i < kFillStages; ++i) {
      mbar_init(&s.fill_full[i], 4);
      mbar_init(&s.fill_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s.acc_full[i], 1);
      mbar_init(&s.acc_empty[i], kWarps);
    }
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(&s.tmem_base, 2 * kColumns);
    tmem_relinquish();
  }
  if (warp == 0 && lane == 0) {
    if (!CODES) tma_prefetch_map(&map_x);
    tma_prefetch_map(&map_dy);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s.tmem_base;
  wait_for_kernel_before();  // the padded copies of the operands, where there are some

  const int quarter = warp & 3, group = warp / 4;  // TMEM lanes 32 quarter.., columns kMine group..
  const uint32_t mine = (static_cast<uint32_t>(quarter * 32) << 16) + group * kMine;
  float acc[kMine];
#pragma unroll
  for (int i = 0; i < kMine; ++i) acc[i] = 0.f;
  int drained = 0;
  bool ok = true;

  // adds the oldest chunk's accumulator to the registers
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
  // A chunk is drained by the time its accumulator is wanted again: before stage `it` is touched, chunks
  // that ended `behind` stages ago are. Their products are (nearly) complete then, so the wait is short,
  // and the other accumulator has products to take meanwhile.
  auto drain_before = [&](int it, int behind) {
    while (ok && it >= (drained + 1) * kChunk + behind) drain();
  };
  if (warp == 0) {
    int it = 0;
    for (; it < steps && ok; ++it) {
      drain_before(it, kStages);
      const int st = it % kStages;
      ok = ok && mbar_wait(&s.empty[st], ((it / kStages) & 1) ^ 1, p.err, kErrTimeoutEmpty);
      ok = __all_sync(0xFFFFFFFFu, ok);
      if (!ok) break;
      if (lane == 0) {
        // panels wholly past the matrix are not loaded (their part of dW is not written)
        const int row = static_cast<int>(first + static_cast<int64_t>(it) * kRows);
        int bytes = 0;
        for (int q = 0; q < BN / 64; ++q) bytes += n0 + 64 * q < p.n ? kPanel : 0;
        if (!CODES)
          for (int q = 0; q < 2 * MB; ++q) bytes += k0 + 64 * q < p.k ? kPanel : 0;
        mbar_arrive_expect_tx(&s.full[st], bytes);
        for (int q = 0; q < BN / 64; ++q)
          if (n0 + 64 * q < p.n) tma_load_2d(s.tma[st] + q * kPanel, &map_dy, &s.full[st], n0 + 64 * q, row);
        if (!CODES)
          for (int q = 0; q < 2 * MB; ++q)
            if (k0 + 64 * q < p.k) tma_load_2d(s.tma[st] + (BN / 64 + q) * kPanel, &map_x, &s.full[st], k0 + 64 * q, row);
      }
      __syncwarp();
    }
    if (!ok && lane == 0) {
      // given up: what was fetched has to land before the CTA may exit (otherwise the drained products show it)
      for (int j = it > kStages ? it - kStages : 0; j < it; ++j)
        mbar_wait(&s.full[j % kStages], (j / kStages) & 1, p.err, kErrTimeoutLoad);
    }
  } else if (warp == 1) {
    const uint32_t idesc = idesc_bf16_f32_abmn(128, BN);
    for (int it = 0; it < steps && ok; ++it) {
      drain_before(it, kChunk / 2);
      const int st = it % kStages, chunk = it / kChunk, fs = it % kFillStages;
      if (ok && it % kChunk == 0) ok = mbar_wait(&s.acc_empty[chunk & 1], ((chunk >> 1) & 1) ^ 1, p.err, kErrTimeoutEmpty);
      ok = ok && mbar_wait(&s.full[st], (it / kStages) & 1, p.err, kErrTimeoutLoad);
      if (CODES) ok = ok && mbar_wait(&s.fill_full[fs], (it / kFillStages) & 1, p.err, kErrTimeoutLoad);
      ok = __all_sync(0xFFFFFFFFu, ok);
      if (!ok) break;
      tc_fence_after();
      if (lane == 0) {
        const uint8_t* x = CODES ? s.fill + fs * (2 * MB * kPanel) : s.tma[st] + BN / 64 * kPanel;
        const uint64_t dx = desc_mnmajor_sw128(smem_u32(x), kPanel, 1024), dd = desc_mnmajor_sw128(smem_u32(s.tma[st]), kPanel, 1024);
        const uint32_t d = tmem + (chunk & 1) * kColumns;
#pragma unroll
        for (int kk = 0; kk < kRows / 16; ++kk) {
          // 16 rows further: two 8-row groups of 1024 bytes (128 in the descriptor's units of 16)
#pragma unroll
          for (int m = 0; m < MB; ++m)
            mma_bf16(d + m * BN, dx + m * (2 * kPanel / 16) + kk * 128, dd + kk * 128, idesc, (it % kChunk | kk) != 0);
        }
        mma_commit(&s.empty[st]);
        if (CODES) mma_commit(&s.fill_empty[fs]);
        if (it % kChunk == kChunk - 1 || it == steps - 1) mma_commit(&s.acc_full[chunk & 1]);
      }
      __syncwarp();
    }
  } else if (CODES && warp >= kWarps - 4 * kGroups) {
    using Rows = CodeRows<2 * MB>;
    const int worker = warp - (kWarps - 4 * kGroups);
    const int of = worker / 4;  // the group: stages of, of + kGroups, ..
    Rows rows(p, k0, first, end, of * kRows + (warp & 3) * kWarpRows, lane);
    uint8_t* const ring = s.ring[worker];
    auto copy = [&](int slot) {
      rows.copy(smem_u32(ring) + slot * Rows::kSlot, p, k0);
      copy_async_commit();
    };
#pragma unroll
    for (int slot = 0; slot < kSlots; ++slot) copy(slot);  // stages past the last: zeros
    int slot = 0;
    for (int it = of; it < steps && ok; it += kGroups) {
      drain_before(it, kFillStages);
      const int fs = it % kFillStages;
      ok = ok && mbar_wait(&s.fill_empty[fs], ((it / kFillStages) & 1) ^ 1, p.err, kErrTimeoutEmpty);
      ok = __all_sync(0xFFFFFFFFu, ok);
      if (!ok) break;
      copy_async_wait<kSlots - 1>();
      __syncwarp();
      rows.fill(s.fill + fs * (2 * MB * kPanel), ring + slot * Rows::kSlot, p);
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&s.fill_full[fs]);
      copy(slot);
      slot = slot == kSlots - 1 ? 0 : slot + 1;
    }
    copy_async_wait<0>();
  }
  while (ok && drained < chunks) drain();
  let_next_kernel_start();
  if (ok) {
    // a lane is a channel of X, a column one of dY: each store of a warp writes 32 neighbours of a row of dW
    const int kk = k0 + (group * kMine / BN) * 128 + quarter * 32 + lane;
    const int nn = n0 + group * kMine % BN;
    if (kk < p.k) {
      float* o = p.out + (static_cast<int64_t>(blockIdx.y) * p.n + nn) * p.k + kk;  // one split: split 0
      if (nn + kMine <= p.n) {
#pragma unroll
        for (int i = 0; i < kMine; ++i, o += p.k) *o = acc[i];
      } else {
#pragma unroll
        for (int i = 0; i < kMine; ++i, o += p.k)
          if (nn + i < p.n) *o = acc[i];
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 2 * kColumns);
  }
}

// ---- operands that neither TMA nor the fill warps take: bf16 rows of a multiple of 8 channels, the last
// ones 0, from bf16 rows of any width or from a checkpoint's (16-byte aligned tensors). A thread writes 8
// channels: it takes the two aligned words (16 bytes, or 8 of codes) that hold them and shifts.
struct PadJob {
  const uint8_t* from;    // bf16 rows, or codes
  const uint8_t* scales;  // null: from bf16
  uint4* out;
  int64_t bytes;          // of `from`
  int width;
  uint32_t total;         // pieces of 8 channels of all rows (0: nothing to do)
  Divisor pieces;         // of a row of `out`
};

// the aligned word at `at`, put together from its elements where the tensor ends inside it
template <typename Word, int SIZE>
__device__ __forceinline__ Word pad_word(const PadJob& j, int64_t at) {
  if (at + static_cast<int64_t>(sizeof(Word)) <= j.bytes) return __ldg(reinterpret_cast<const Word*>(j.from + at));
  uint32_t w[sizeof(Word) / 4] = {};
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(Word)); i += SIZE)
    if (at + i < j.bytes) {
      const uint32_t e = SIZE == 1 ? static_cast<uint32_t>(__ldg(j.from + at + i))
                                   : static_cast<uint32_t>(__ldg(reinterpret_cast<const uint16_t*>(j.from + at + i)));
      w[i / 4] |= e << (8 * (i & 3));
    }
  Word out;
  memcpy(&out, w, sizeof(out));
  return out;
}

__global__ void __launch_bounds__(256) wgrad_pad_kernel(PadJob first, PadJob second) {
  for (int which = 0; which < 2; ++which) {
    const PadJob& j = which == 0 ? first : second;
    const int blocks = (j.width + kMxBlock - 1) / kMxBlock;
    for (uint32_t id = blockIdx.x * 256 + threadIdx.x; id < j.total; id += gridDim.x * 256) {
      const uint32_t row = j.pieces.quotient(id);
      const int col = static_cast<int>(id - row * j.pieces.d) * 8;
      const int left = j.width - col;  // channels there are: the others become 0
      const int64_t at = static_cast<int64_t>(row) * j.width + col;
      uint4 v;
      if (j.scales == nullptr) {
        const uint32_t shift = static_cast<uint32_t>(2 * at) & 15u;
        const uint4 lo = pad_word<uint4, 2>(j, 2 * at - shift), hi = pad_word<uint4, 2>(j, 2 * at - shift + 16);
        uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
        for (int i = 0; i < 6; ++i) w[i] = shift & 8u ? w[i + 2] : w[i];
#pragma unroll
        for (int i = 0; i < 5; ++i) w[i] = shift & 4u ? w[i + 1] : w[i];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], (shift & 2u) * 8);
        v = make_uint4(w[0], w[1], w[2], w[3]);
      } else {
        const uint32_t shift = static_cast<uint32_t>(at) & 7u;
        const uint2 lo = pad_word<uint2, 1>(j, at - shift), hi = pad_word<uint2, 1>(j, at - shift + 8);
        const uint32_t w0 = shift & 4u ? lo.y : lo.x, w1 = shift & 4u ? hi.x : lo.y, w2 = shift & 4u ? hi.y : hi.x;
        const uint2 c = make_uint2(__funnelshift_r(w0, w1, (shift & 3u) * 8), __funnelshift_r(w1, w2, (shift & 3u) * 8));
        v = mx_decode_bf16(c, __ldg(j.scales + static_cast<int64_t>(row) * blocks + col / kMxBlock));
      }
      if (left < 8) {
        uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = left >= 2 * i + 2 ? w[i] : left == 2 * i + 1 ? w[i] & 0xFFFFu : 0u;
        v = make_uint4(w[0], w[1], w[2], w[3]);
      }
      j.out[id] = v;
    }
  }
}

// dW = the splits' partial sums [split][n k], added in a fixed order: a thread takes VEC elements of every
// GROUPSth split, then the groups' sums of a place are added in turn.
template <int VEC, int GROUPS>
__global__ void __launch_bounds__(256)
    wgrad_reduce_kernel(const float* __restrict__ part, float* __restrict__ out, int splits, int64_t count) {
  constexpr int kPlaces = 256 / GROUPS;
  __shared__ float sum[GROUPS][kPlaces * VEC];
  const int place = threadIdx.x % kPlaces, g = threadIdx.x / kPlaces;
  const int64_t at = (static_cast<int64_t>(blockIdx.x) * kPlaces + place) * VEC;
  float a[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) a[i] = 0.f;
  wait_for_kernel_before();
  if (at < count) {
    const float* p = part + at;
#pragma unroll 4
    for (int s = g; s < splits; s += GROUPS) {
      if constexpr (VEC == 4) {
        const float4 v = __ldcs(reinterpret_cast<const float4*>(p + s * count));
        a[0] += v.x;
        a[1] += v.y;
        a[2] += v.z;
        a[3] += v.w;
      } else {
        a[0] += __ldcs(p + s * count);
      }
    }
  }
  if constexpr (GROUPS > 1) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) sum[g][i * kPlaces + place] = a[i];
    __syncthreads();
    if (g != 0) return;
#pragma unroll
    for (int k = 1; k < GROUPS; ++k)
#pragma unroll
      for (int i = 0; i < VEC; ++i) a[i] += sum[k][i * kPlaces + place];
  }
  if (at < count) {
    if constexpr (VEC == 4)
      *reinterpret_cast<float4*>(out + at) = make_float4(a[0], a[1], a[2], a[3]);
    else
      out[at] = a[0];
  }
}

// Many splits are shared out over the block's groups of threads (a place's sum would wait for one load after
// another), few are added by one thread.
template <int VEC, int GROUPS>
int launch_reduce(const float* part, float* out, int splits, int64_t count, cudaStream_t stream) {
  constexpr int places = 256 / GROUPS * VEC;
  return launch_after(wgrad_reduce_kernel<VEC, GROUPS>, static_cast<unsigned>((count + places - 1) / places), 256, 0, stream, part,
                      out, splits, count);
}
template <int VEC>
int launch_reduce(const float* part, float* out, int splits, int64_t count, cudaStream_t stream) {
  return splits > 32  ? launch_reduce<VEC, 32>(part, out, splits, count, stream)
         : splits > 8 ? launch_reduce<VEC, 8>(part, out, splits, count, stream)
                      : launch_reduce<VEC, 1>(part, out, splits, count, stream);
}

struct WgradPlan {
  int mb, bn, tiles, splits;
  int64_t split_rows;
};

// Tiles of 256 channels of dY by 128 of X, or 128 by 256 for few of dY: larger tiles read each operand less
// often.
WgradPlan plan(int64_t rows, int n, int k, bool pad, bool codes) {
  WgradPlan p;
  p.bn = n <= 64 ? 64 : n <= 128 ? 128 : 256;
  p.mb = p.bn == 256 || k <= 128 ? 1 : 2;
  const int64_t tiles = static_cast<int64_t>((n + p.bn - 1) / p.bn) * ((k + 128 * p.mb - 1) / (128 * p.mb));
  p.tiles = static_cast<int>(tiles);
  // The number of splits that ends first, in stages' time: waves of CTAs, each with its own start and end
  // (about 6 stages), and for the partial sums a pass over them (1 for 2^20 sums) and a second kernel, which
  // starts while the products end: 1 stage of an 8-bit X (0.7 us), 3 of the shorter ones of a bf16 X (0.5 us),
  // and 8 beside a padding kernel, where the host's third launch is what a short call waits for. Against 8 in
  // each case, calls issued back to back, 8 bits: 1024 rows, n 1536, k 384 in 13.7 us for 18.5, 512 rows, n 512,
  // k 128 in 10.3 for 13.1. With 1 in each case 512 rows, n 558, k 11 took 11.6 us for 10.5, and 512 rows,
  // n = k = 1024 in bf16 up to 11.4 for 10.3.
  const int second = pad ? 8 : codes ? 1 : 3;
  const int64_t steps = (rows + kRows - 1) / kRows;
  int64_t best = 1, best_cost = -1;
  for (int64_t s = 1; s <= kSms && s <= steps; ++s) {
    if (s > 1 && tiles * s > 4 * kSms) break;  // enough tiles to fill the SMs
    const int64_t waves = (tiles * s + kSms - 1) / kSms;
    const int64_t cost = waves * ((steps + s - 1) / s + 6) + (s > 1 ? second + s * n * k / (1 << 20) : 0);
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

template <int MB, int BN, bool CODES>
int launch(const CUtensorMap& x, const CUtensorMap& dy, const WgradParams& p, const WgradPlan& plan, bool after, cudaStream_t stream) {
  constexpr size_t smem = sizeof(WgradSmem<MB, BN, CODES>) + 1024;
  static_assert(smem <= 232448, "weight-gradient shared memory exceeds the per-CTA limit");
  auto kernel = wgrad_kernel<MB, BN, CODES>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
  if (e != cudaSuccess) return static_cast<int>(e);
  const dim3 grid(plan.tiles, plan.splits);
  if (after) return launch_after(kernel, grid, kWgradThreads, smem, stream, x, dy, p);
  kernel<<<grid, kWgradThreads, smem, stream>>>(x, dy, p);
  return static_cast<int>(cudaGetLastError());
}

template <bool CODES>
int launch_tile(const CUtensorMap& x, const CUtensorMap& dy, const WgradParams& p, const WgradPlan& plan, bool after,
                cudaStream_t s) {
  if (plan.bn == 256) return launch<1, 256, CODES>(x, dy, p, plan, after, s);
  if (plan.mb == 2) return plan.bn == 64 ? launch<2, 64, CODES>(x, dy, p, plan, after, s) : launch<2, 128, CODES>(x, dy, p, plan, after, s);
  return plan.bn == 64 ? launch<1, 64, CODES>(x, dy, p, plan, after, s) : launch<1, 128, CODES>(x, dy, p, plan, after, s);
}

int panel_map(CUtensorMap* map, const void* base, int64_t rows, int width, int pitch) {
  const uint64_t dims[2] = {static_cast<uint64_t>(width), static_cast<uint64_t>(rows)};
  const uint64_t strides[1] = {static_cast<uint64_t>(pitch) * 2};
  const uint32_t box[2] = {64, kRows};
  return make_map(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, base, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
int padded(int width) { return (width + 7) / 8 * 8; }
size_t partial_bytes(const WgradPlan& p, int n, int k) {
  return p.splits > 1 ? (static_cast<size_t>(p.splits) * n * k * sizeof(float) + 255) / 256 * 256 : 0;
}
size_t pad_bytes(int64_t rows, int width) { return (static_cast<size_t>(rows) * padded(width) * 2 + 255) / 256 * 256; }

}  // namespace

size_t weight_grad_workspace_bytes(int64_t rows, int n, int k, bool codes) {
  const bool pad_dy = n % 8 != 0, pad_x = k % (codes ? 16 : 8) != 0;
  size_t bytes = partial_bytes(plan(rows, n, k, pad_dy || pad_x, codes), n, k);
  if (pad_dy) bytes += pad_bytes(rows, n);
  if (pad_x) bytes += pad_bytes(rows, k);
  return bytes;
}

int weight_grad_forward(const void* dy, const void* x, const uint8_t* codes, const uint8_t* scales, float* dw,
                        void* workspace, int64_t rows, int n, int k, const DeviceInfo& info, cudaStream_t stream) {
  const bool pad_dy = n % 8 != 0, pad_x = k % (codes != nullptr ? 16 : 8) != 0;
  const WgradPlan pl = plan(rows, n, k, pad_dy || pad_x, codes != nullptr);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  uint8_t* pad = ws + partial_bytes(pl, n, k);
  const void* const from_dy = dy;
  const void* const from_x = codes != nullptr ? static_cast<const void*>(codes) : x;
  const uint8_t* const from_scales = codes != nullptr ? scales : nullptr;
  uint8_t *pad_for_dy = nullptr, *pad_for_x = nullptr;
  if (pad_dy) {
    dy = pad_for_dy = pad;
    pad += pad_bytes(rows, n);
  }
  if (pad_x) {
    x = pad_for_x = pad;
    codes = nullptr;
  }
  int rc = 0;
  if (pad_dy || pad_x) {
    // so many rows at a time that their pieces are counted in 31 bits; a multiple of 16, so that each piece
    // of a tensor starts on a 16-byte boundary
    const int64_t most = (int64_t(1) << 30) / (padded(n > k ? n : k) / 8) / 16 * 16;
    for (int64_t first = 0; first < rows && rc == 0; first += most) {
      const int64_t part = rows - first < most ? rows - first : most;
      auto job = [&](const void* from, const uint8_t* s, uint8_t* out, int width) {
        const int pieces = padded(width) / 8, size = s != nullptr ? 1 : 2;
        return PadJob{static_cast<const uint8_t*>(from) + first * width * size,
                      s != nullptr ? s + first * ((width + kMxBlock - 1) / kMxBlock) : nullptr,
                      out != nullptr ? reinterpret_cast<uint4*>(out) + first * pieces : nullptr,
                      part * width * size,
                      width,
                      out != nullptr ? static_cast<uint32_t>(part * pieces) : 0u,
                      Divisor(static_cast<uint32_t>(pieces))};
      };
      const PadJob a = job(from_dy, nullptr, pad_for_dy, n), b = job(from_x, from_scales, pad_for_x, k);
      const uint32_t blocks = ((a.total > b.total ? a.total : b.total) + 255) / 256;
      wgrad_pad_kernel<<<blocks < 148 * 16 ? blocks : 148 * 16, 256, 0, stream>>>(a, b);
      rc = static_cast<int>(cudaGetLastError());
    }
    if (rc != 0) return cuda_status(rc, "weight_grad launch");
  }
  CUtensorMap mx, md;
  memset(&mx, 0, sizeof(mx));
  int st = panel_map(&md, dy, rows, n, padded(n));
  if (st == 0 && codes == nullptr) st = panel_map(&mx, x, rows, k, padded(k));
  if (st != 0) return st;
  WgradParams p;
  p.codes = codes;
  p.scales = scales;
  p.rows = rows;
  p.split_rows = pl.split_rows;
  p.n = n;
  p.k = k;
  p.out = pl.splits > 1 ? reinterpret_cast<float*>(ws) : dw;
  p.err = info.err;
  const bool after = pad_dy || pad_x;
  rc = codes != nullptr ? launch_tile<true>(mx, md, p, pl, after, stream) : launch_tile<false>(mx, md, p, pl, after, stream);
  if (rc == 0 && pl.splits > 1) {
    const int64_t count = static_cast<int64_t>(n) * k;
    const float* part = reinterpret_cast<const float*>(ws);
    rc = count % 4 == 0 && aligned16(dw) ? launch_reduce<4>(part, dw, pl.splits, count, stream)
                                         : launch_reduce<1>(part, dw, pl.splits, count, stream);
  }
  return cuda_status(rc, "weight_grad launch");
}

}  // namespace ffb
