// Weight preparation: fp32 master weights -> bf16 tensor-core operands.
//
// A LayerNorm followed by a projection, W (gamma * xhat + beta), is applied to the RAW
// activation x as  rstd * (W' x - mean * wsum) + bias  with
//   W'   = bf16(W diag(gamma))       the MMA operand,
//   wsum = sum_k W'[n, k]            (of the bf16-rounded W', so the subtraction is exact
//                                     with respect to what the tensor core multiplied),
//   bias = W beta                    (fp32),
// so the kernels feed raw bf16 activations straight from TMA to the tensor core and the
// normalisation costs two FMAs per output in the epilogue.
//
// The operand is written in the shared-memory image the kernels use: K-major, 64-column
// (128-byte) blocks of `rows` rows each, 16-byte chunks XOR-swizzled by (row % 8). A
// kernel copies the image linearly into 1024-byte aligned shared memory.
#include "common.cuh"
#include "kernels.h"

namespace ffb {
namespace {

// A block packs kPackRows rows, kPackColumns of each at a time: all threads write the image, then one thread a
// row and sum adds up the columns in turn from shared memory (wsum and bias have that order). A pair transition, which
// a training step packs in every forward pass, is packed in 72 us; with one thread for the whole of a row
// it took 411.
constexpr int kPackRows = 8, kPackColumns = 128;

__global__ void __launch_bounds__(kPackColumns)
    pack_weight_kernel(const float* __restrict__ w, int rows, int k, const float* __restrict__ gamma,
                       const float* __restrict__ beta, uint8_t* __restrict__ image, int row_offset, int image_rows,
                       float* __restrict__ wsum, float* __restrict__ bias, float scale) {
  __shared__ float packed[kPackRows][kPackColumns + 1], plain[kPackRows][kPackColumns + 1], shift[kPackColumns];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int first = blockIdx.x * kPackRows;
  const int here = rows - first < kPackRows ? rows - first : kPackRows;
  float s = 0.f, bsum = 0.f;
  for (int c0 = 0; c0 < k; c0 += kPackColumns) {
    const int n = k - c0 < kPackColumns ? k - c0 : kPackColumns, j = threadIdx.x, c = c0 + j;
    if (j < n) {  // a thread has the same column of every row
      const float g = gamma ? gamma[c] : 1.0f;
      uint8_t* block = image + static_cast<int64_t>(c / 64) * image_rows * 128;
      shift[j] = beta ? beta[c] : 0.f;
      float v[kPackRows];
#pragma unroll
      for (int r = 0; r < kPackRows; ++r) v[r] = r < here ? w[static_cast<int64_t>(first + r) * k + c] : 0.f;
#pragma unroll
      for (int r = 0; r < kPackRows; ++r) {
        if (r >= here) break;
        const __nv_bfloat16 q = __float2bfloat16_rn(v[r] * g * scale);
        *reinterpret_cast<__nv_bfloat16*>(block + sw128_offset(row_offset + first + r, c % 64)) = q;
        packed[r][j] = __bfloat162float(q);
        plain[r][j] = v[r];
      }
    }
    __syncthreads();
    if (warp == 0 && lane < here && wsum) {
#pragma unroll 16
      for (int j = 0; j < n; ++j) s += packed[lane][j];
    }
    if (warp == 1 && lane < here && bias && beta) {
#pragma unroll 16
      for (int j = 0; j < n; ++j) bsum += plain[lane][j] * shift[j];
    }
    __syncthreads();
  }
  if (warp == 0 && lane < here && wsum) wsum[row_offset + first + lane] = s;
  if (warp == 1 && lane < here && bias) bias[row_offset + first + lane] = bsum * scale;
}

}  // namespace

int launch_pack_weight(const float* w, int rows, int k, const float* gamma, const float* beta, uint8_t* image,
                       int row_offset, int image_rows, float* wsum, float* bias, cudaStream_t stream, float scale) {
  pack_weight_kernel<<<(rows + kPackRows - 1) / kPackRows, kPackColumns, 0, stream>>>(
      w, rows, k, gamma, beta, image, row_offset, image_rows, wsum, bias, scale);
  return static_cast<int>(cudaGetLastError());
}

}  // namespace ffb
