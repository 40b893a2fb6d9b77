// A linear layer's weight gradient dW [n, k] = dY^T X over `rows` rows, fp32 sums and output:
// dY [rows, n] bf16, X [rows, k] bf16 or its 8-bit checkpoint (mx8.cuh).
//
// The reduction runs along the rows, so both operands are MN-major for tcgen05: 64 rows of 64
// channels are one 128-byte-swizzled panel of 8 KB, exactly what a TMA box of a row-major tensor
// leaves in shared memory. An 8-bit X is turned into bf16 on the way into shared memory (e4m3 times a
// power of two fits bf16's 8 bits of mantissa, so nothing is lost) and never exists in global memory.
//
// A pair tensor has rows = N^2 and n, k of a few hundred: few output tiles and a long reduction, so
// the rows are split over the SMs. A CTA takes one (128 MB) x BN tile of dW and one range of rows and
// leaves its fp32 sums in the workspace; wgrad_reduce_kernel adds the ranges in a fixed order.
#include <string.h>

#include "abi_util.h"
#include "common.cuh"
#include "kernels.h"
#include "mx8.cuh"

namespace ffb {
namespace {

constexpr int kRows = 64;                  // rows (the K of the product) of a stage
constexpr int kPanel = kRows * 128;        // bytes of a panel: 64 rows x 64 bf16 channels
constexpr int kLoaders = 8;                // loader / epilogue warps
constexpr int kWgradThreads = 64 + 32 * kLoaders;
constexpr int kTargetCtas = 148;           // one CTA an SM; fixed, so that a result does not depend on the device's SM count

struct WgradParams {
  const __nv_bfloat16* dy;
  const __nv_bfloat16* x;
  const uint8_t* codes;
  const uint8_t* scales;
  float* out;       // dW, or the workspace of partial sums
  int64_t rows;
  int64_t split_rows;  // rows of a split, a multiple of kRows
  int n, k;
  int partial;      // leave partial sums instead of dW
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
  uint64_t done;
  uint32_t tmem_base;
};

// Both operands MN-major, bf16 -> fp32.
__host__ __device__ constexpr uint32_t idesc_bf16_f32_abmn(int m, int n) {
  return idesc_bf16_f32(m, n) | (1u << 15) | (1u << 16);
}

// Eight consecutive elements of a row as bf16, 0 past the tensor's end: any alignment.
__device__ __forceinline__ uint4 load8_any(const __nv_bfloat16* p, int left) {
  uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < left) w[i / 2] |= static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(p + i)) << (16 * (i & 1));
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Fills `panels` panels with rows [row0, row0 + 64) and channels [col0, col0 + 64 panels) of a bf16
// matrix of any alignment; rows past `end` and channels past `width` are 0.
__device__ __forceinline__ void fill_any(uint8_t* dst, const __nv_bfloat16* src, int panels, int64_t row0, int64_t end,
                                         int col0, int width, int id) {
  for (int q = id; q < panels * kRows * 8; q += 32 * kLoaders) {
    const int chunk = q & 7, panel = (q >> 3) % panels, r = q / (8 * panels);
    const int64_t row = row0 + r;
    const int col = col0 + panel * 64 + chunk * 8;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (row < end && col < width) v = load8_any(src + row * width + col, width - col);
    *reinterpret_cast<uint4*>(dst + panel * kPanel + sw128_offset(r, chunk * 8)) = v;
  }
}

// The same from an 8-bit checkpoint: eight codes a step (one load where the rows allow it).
__device__ __forceinline__ void fill_codes(uint8_t* dst, const uint8_t* codes, const uint8_t* scales, int panels,
                                           int64_t row0, int64_t end, int col0, int width, bool vector, int id) {
  const int blocks = (width + kMxBlock - 1) / kMxBlock;
  for (int q = id; q < panels * kRows * 8; q += 32 * kLoaders) {
    const int chunk = q & 7, panel = (q >> 3) % panels, r = q / (8 * panels);
    const int64_t row = row0 + r;
    const int col = col0 + panel * 64 + chunk * 8;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (row < end && col < width) {
      uint2 c = make_uint2(0, 0);
      const uint8_t* p = codes + row * width + col;
      if (vector) {
        c = *reinterpret_cast<const uint2*>(p);
      } else {
        uint32_t w[2] = {0, 0};
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (i < width - col) w[i / 4] |= static_cast<uint32_t>(p[i]) << (8 * (i & 3));
        c = make_uint2(w[0], w[1]);
      }
      float f[8];
      mx_decode<8>(c, mx_scale(scales[row * blocks + col / kMxBlock]), f);
      v = make_uint4(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]), pack_bf16(f[4], f[5]), pack_bf16(f[6], f[7]));
    }
    *reinterpret_cast<uint4*>(dst + panel * kPanel + sw128_offset(r, chunk * 8)) = v;
  }
}

// A_TMA / B_TMA: the operand's panels come by TMA (bf16 rows of a multiple of 8 channels, 16-byte
// aligned); otherwise the loader warps fill them. MX: X is a checkpoint (always filled).
template <int MB, int BN, bool A_TMA, bool B_TMA, bool MX>
__global__ void __launch_bounds__(kWgradThreads, 1)
    wgrad_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, WgradParams p) {
  using Smem = WgradSmem<MB, BN>;
  constexpr int kStages = Smem::kStages;
  constexpr int kColumns = MB * BN;  // TMEM columns: a power of two, 64 to 512
  constexpr bool kFill = !A_TMA || !B_TMA;
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
      mbar_init(&s.full[i], (A_TMA || B_TMA ? 1 : 0) + (kFill ? kLoaders : 0));
      mbar_init(&s.empty[i], 1);
    }
    mbar_init(&s.done, 1);
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(&s.tmem_base, kColumns);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s.tmem_base;

  if (warp == 0) {
    if ((A_TMA || B_TMA) && lane == 0) {
      int it = 0;
      for (; it < steps; ++it) {
        const int st = it % kStages;
        if (!mbar_wait(&s.empty[st], ((it / kStages) & 1) ^ 1, p.err, kErrTimeoutEmpty)) break;
        const int row = static_cast<int>(first + static_cast<int64_t>(it) * kRows);
        // panels wholly past the matrix are not loaded (their columns of dW are not written)
        int bytes = 0;
        if (A_TMA)
          for (int q = 0; q < 2 * MB; ++q) bytes += n0 + 64 * q < p.n ? kPanel : 0;
        if (B_TMA)
          for (int q = 0; q < BN / 64; ++q) bytes += k0 + 64 * q < p.k ? kPanel : 0;
        mbar_arrive_expect_tx(&s.full[st], bytes);
        if (A_TMA)
          for (int q = 0; q < 2 * MB; ++q)
            if (n0 + 64 * q < p.n) tma_load_2d(s.a[st] + q * kPanel, &map_a, &s.full[st], n0 + 64 * q, row);
        if (B_TMA)
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
      bool ok = true;
      for (int it = 0; it < steps; ++it) {
        const int st = it % kStages;
        if (!mbar_wait(&s.full[st], (it / kStages) & 1, p.err, kErrTimeoutLoad)) { ok = false; break; }
        tc_fence_after();
        const uint32_t a = smem_u32(s.a[st]), b = smem_u32(s.b[st]);
#pragma unroll
        for (int kk = 0; kk < kRows / 16; ++kk) {
          // 16 rows further: two 8-row groups of 1024 bytes
          const uint64_t db = desc_mnmajor_sw128(b + kk * 2048, kPanel, 1024);
#pragma unroll
          for (int m = 0; m < MB; ++m)
            mma_bf16(tmem + m * BN, desc_mnmajor_sw128(a + m * 2 * kPanel + kk * 2048, kPanel, 1024), db, idesc,
                     (it | kk) != 0);
        }
        mma_commit(&s.empty[st]);
      }
      if (ok) mma_commit(&s.done);
    }
  } else {
    const int id = threadIdx.x - 64;
    bool ok = true;
    if (kFill) {
      for (int it = 0; it < steps; ++it) {
        const int st = it % kStages;
        const int64_t row = first + static_cast<int64_t>(it) * kRows;
        ok = mbar_wait(&s.empty[st], ((it / kStages) & 1) ^ 1, p.err, kErrTimeoutEmpty);
        if (!ok) break;
        if (!A_TMA) fill_any(s.a[st], p.dy, 2 * MB, row, end, n0, p.n, id);
        if (!B_TMA) {
          if (MX)
            fill_codes(s.b[st], p.codes, p.scales, BN / 64, row, end, k0, p.k, p.k % 8 == 0, id);
          else
            fill_any(s.b[st], p.x, BN / 64, row, end, k0, p.k, id);
        }
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s.full[st]);
      }
    }
    ok = ok && mbar_wait(&s.done, 0, p.err, kErrTimeoutMma);
    ok = __all_sync(0xFFFFFFFFu, ok);
    if (ok) {
      tc_fence_after();
      // eight warps: TMEM lane quarter = warp % 4; the two warps of a quarter take half of the columns each
      const int quarter = warp & 3, half = (warp - 2) / 4;
      for (int c = half * (kColumns / 2); c < (half + 1) * (kColumns / 2); c += 32) {
        __syncwarp();
        uint32_t v[32];
        tmem_ld32(tmem + (static_cast<uint32_t>(quarter * 32) << 16) + c, v);
        tmem_ld_wait();
        const int nn = n0 + (c / BN) * 128 + quarter * 32 + lane;
        const int kk = k0 + c % BN;
        if (nn >= p.n || kk >= p.k) continue;
        float* o = p.out + (p.partial ? static_cast<int64_t>(blockIdx.y) * p.n * p.k : 0) +
                   static_cast<int64_t>(nn) * p.k + kk;
        if (kk + 32 <= p.k && (reinterpret_cast<uintptr_t>(o) & 15u) == 0) {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            reinterpret_cast<uint4*>(o)[i] = make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (kk + i < p.k) o[i] = __uint_as_float(v[i]);
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, kColumns);
  }
}

// dW = the splits' partial sums, added in a fixed order.
__global__ void __launch_bounds__(256) wgrad_reduce_kernel(const float* __restrict__ part, float* __restrict__ out,
                                                            int64_t count, int splits) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= count) return;
  float a = 0.f;
#pragma unroll 8
  for (int s = 0; s < splits; ++s) a += part[s * count + i];
  out[i] = a;
}

struct WgradPlan {
  int mb, bn, tiles, splits;
  int64_t split_rows;
};

WgradPlan plan(int64_t rows, int n, int k) {
  WgradPlan p;
  p.mb = n <= 128 ? 1 : 2;
  // 256 columns a tile where that pads dW no further than 128 would
  p.bn = k <= 64 ? 64 : (k + 255) / 256 * 2 <= (k + 127) / 128 ? 256 : 128;
  const int64_t tiles = static_cast<int64_t>((n + 128 * p.mb - 1) / (128 * p.mb)) * ((k + p.bn - 1) / p.bn);
  p.tiles = static_cast<int>(tiles);
  const int64_t steps = (rows + kRows - 1) / kRows;
  int64_t splits = kTargetCtas / tiles;
  if (splits > steps / 2) splits = steps / 2;  // at least two stages a split
  if (splits < 1) splits = 1;
  const int64_t per = (steps + splits - 1) / splits;
  p.split_rows = per * kRows;
  p.splits = static_cast<int>((steps + per - 1) / per);  // no empty split
  return p;
}

template <int MB, int BN, bool A_TMA, bool B_TMA, bool MX>
int launch(const CUtensorMap& a, const CUtensorMap& b, const WgradParams& p, const WgradPlan& plan, cudaStream_t stream) {
  constexpr size_t smem = sizeof(WgradSmem<MB, BN>) + 1024;
  static_assert(smem <= 232448, "weight-gradient shared memory exceeds the per-CTA limit");
  auto kernel = wgrad_kernel<MB, BN, A_TMA, B_TMA, MX>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
  if (e != cudaSuccess) return static_cast<int>(e);
  kernel<<<dim3(plan.tiles, plan.splits), kWgradThreads, smem, stream>>>(a, b, p);
  return static_cast<int>(cudaGetLastError());
}

template <int MB, int BN>
int launch_operands(const CUtensorMap& a, const CUtensorMap& b, const WgradParams& p, const WgradPlan& plan, bool a_tma,
                    bool b_tma, cudaStream_t stream) {
  if (p.codes != nullptr)
    return a_tma ? launch<MB, BN, true, false, true>(a, b, p, plan, stream)
                 : launch<MB, BN, false, false, true>(a, b, p, plan, stream);
  if (a_tma)
    return b_tma ? launch<MB, BN, true, true, false>(a, b, p, plan, stream)
                 : launch<MB, BN, true, false, false>(a, b, p, plan, stream);
  return b_tma ? launch<MB, BN, false, true, false>(a, b, p, plan, stream)
               : launch<MB, BN, false, false, false>(a, b, p, plan, stream);
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
  const WgradPlan p = plan(rows, n, k);
  return p.splits > 1 ? static_cast<size_t>(p.splits) * n * k * sizeof(float) : 0;
}

int weight_grad_forward(const void* dy, const void* x, const uint8_t* codes, const uint8_t* scales, float* dw,
                        void* workspace, int64_t rows, int n, int k, const DeviceInfo& info, cudaStream_t stream) {
  const WgradPlan pl = plan(rows, n, k);
  const bool a_tma = by_tma(dy, n), b_tma = codes == nullptr && by_tma(x, k);
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
  if (pl.mb == 1)
    rc = pl.bn == 64    ? launch_operands<1, 64>(ma, mb, p, pl, a_tma, b_tma, stream)
         : pl.bn == 128 ? launch_operands<1, 128>(ma, mb, p, pl, a_tma, b_tma, stream)
                        : launch_operands<1, 256>(ma, mb, p, pl, a_tma, b_tma, stream);
  else
    rc = pl.bn == 64    ? launch_operands<2, 64>(ma, mb, p, pl, a_tma, b_tma, stream)
         : pl.bn == 128 ? launch_operands<2, 128>(ma, mb, p, pl, a_tma, b_tma, stream)
                        : launch_operands<2, 256>(ma, mb, p, pl, a_tma, b_tma, stream);
  if (rc == 0 && p.partial) {
    const int64_t count = static_cast<int64_t>(n) * k;
    wgrad_reduce_kernel<<<static_cast<int>((count + 255) / 256), 256, 0, stream>>>(static_cast<const float*>(workspace),
                                                                                   dw, count, pl.splits);
    rc = static_cast<int>(cudaGetLastError());
  }
  return cuda_status(rc, "weight_grad launch");
}

}  // namespace ffb
