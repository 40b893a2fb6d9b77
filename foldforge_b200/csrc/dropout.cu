// Dropout from a counter-based generator: an update dropped, scaled and added to its residual in one pass.
// The mask is never stored: an element's word follows from the seed and the element's number alone, so the
// backward pass draws it again, and neither the grid nor a tensor's layout enters it.
#include "kernels.h"
#include "launch.cuh"
#include "mx8.cuh"

namespace ffb {
namespace {

constexpr int kThreads = 256;

// Philox4x32-10: J. Salmon, M. Moraes, R. Dror and D. Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011.
__device__ __forceinline__ uint4 philox(uint64_t counter, uint64_t offset, uint64_t seed) {
  uint32_t c0 = static_cast<uint32_t>(counter), c1 = static_cast<uint32_t>(counter >> 32);
  uint32_t c2 = static_cast<uint32_t>(offset), c3 = static_cast<uint32_t>(offset >> 32);
  uint32_t k0 = static_cast<uint32_t>(seed), k1 = static_cast<uint32_t>(seed >> 32);
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t p0 = static_cast<uint64_t>(c0) * 0xD2511F53u, p1 = static_cast<uint64_t>(c2) * 0xCD9E8D57u;
    c0 = static_cast<uint32_t>(p1 >> 32) ^ c1 ^ k0;
    c1 = static_cast<uint32_t>(p1);
    c2 = static_cast<uint32_t>(p0 >> 32) ^ c3 ^ k1;
    c3 = static_cast<uint32_t>(p0);
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return make_uint4(c0, c1, c2, c3);
}

template <typename TX, typename TO>
__global__ void __launch_bounds__(kThreads) dropout_kernel(const DropoutParams p, int64_t total) {
  uint64_t seed = p.seed, offset = p.offset;
  if (p.device_seed != nullptr) {
    seed = p.device_seed[0];
    offset += p.device_seed[1];
  }
  const TX* x = static_cast<const TX*>(p.x);
  const TO* residual = static_cast<const TO*>(p.residual);
  TO* out = static_cast<TO*>(p.out);
  for (int64_t i = blockIdx.x * static_cast<int64_t>(kThreads) + threadIdx.x; i < total;
       i += static_cast<int64_t>(gridDim.x) * kThreads) {
    const int64_t row = i / p.inner, m = row / p.shared * p.inner + (i - row * p.inner);
    const uint4 words = philox(static_cast<uint64_t>(m) / 4, offset, seed);
    const uint32_t word = (m & 2) != 0 ? ((m & 1) != 0 ? words.w : words.z) : ((m & 1) != 0 ? words.y : words.x);
    float v = word >= p.threshold ? static_cast<float>(x[i]) * p.scale : 0.f;
    if (residual != nullptr) v += static_cast<float>(residual[i]);
    out[i] = static_cast<TO>(v);
  }
}

template <typename TX, typename TO>
int dropout(const DropoutParams& p, cudaStream_t stream) {
  const int64_t total = p.outer * p.shared * p.inner, want = (total + kThreads - 1) / kThreads;
  dropout_kernel<TX, TO><<<static_cast<unsigned>(want < 148 * 64 ? want : 148 * 64), kThreads, 0, stream>>>(p, total);
  return static_cast<int>(cudaGetLastError());
}

}  // namespace

int launch_dropout(const DropoutParams& p, int x_is_f32, int out_is_f32, cudaStream_t stream) {
  if (x_is_f32) return out_is_f32 ? dropout<float, float>(p, stream) : dropout<float, __nv_bfloat16>(p, stream);
  return out_is_f32 ? dropout<__nv_bfloat16, float>(p, stream) : dropout<__nv_bfloat16, __nv_bfloat16>(p, stream);
}

}  // namespace ffb
