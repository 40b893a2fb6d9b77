// Small helpers around launches: division by a number fixed per launch, and kernels that start while the
// one before them ends.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace ffb {

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

// ---- programmatic dependent launch: a kernel launched with launch_after may start (its blocks take their
// places, its set-up runs) once every block of the kernel before it in the stream has called
// let_next_kernel_start or ended. What that kernel wrote may be read after wait_for_kernel_before, which
// waits for its end; every thread that reads or writes memory calls it first. Against launches after that
// end, calls issued back to back: LayerNorm steps 0.7 to 2.2 us shorter (262144 x 128 with a checkpoint 72.6
// -> 71.9, 4099 x 4096 53.5 -> 51.3), weight gradients 2 us (66.4 -> 64.4), with padded rows 3 to 5 (34.4 ->
// 29.6 to 31.1).
__device__ __forceinline__ void let_next_kernel_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_kernel_before() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

template <typename... Params, typename... Args>
int launch_after(void (*kernel)(Params...), dim3 grid, int threads, size_t smem, cudaStream_t stream, Args... args) {
  cudaLaunchAttribute attribute;
  attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config = {};
  config.gridDim = grid;
  config.blockDim = dim3(static_cast<unsigned>(threads));
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  config.attrs = &attribute;
  config.numAttrs = 1;
  return static_cast<int>(cudaLaunchKernelEx(&config, kernel, static_cast<Params>(args)...));
}

}  // namespace ffb
