// The C ABI of the training operators: argument checks around train.cu and wgrad.cu.
#include "../../include/foldforge_b200.h"
#include "abi_util.h"
#include "kernels.h"

using namespace ffb;

namespace {

// what every entry point here asks of its sizes and its dtype
int check_rows(const char* what, int64_t rows, int64_t c, int dtype) {
  if (rows < 0 || c <= 0) return fail(FFB_ERR_ARG, "%s: rows=%lld c=%lld", what, (long long)rows, (long long)c);
  if (c > (1 << 30)) return fail(FFB_ERR_UNSUPPORTED, "%s: %lld channels", what, (long long)c);
  if (rows > (int64_t(1) << 46) / c) return fail(FFB_ERR_UNSUPPORTED, "%s: too many elements", what);
  if (dtype != FFB_BF16 && dtype != FFB_F32) return fail(FFB_ERR_UNSUPPORTED, "%s: dtype %d", what, dtype);
  return FFB_OK;
}

int element_size(int dtype) { return dtype == FFB_F32 ? 4 : 2; }

// an element-aligned pointer (the kernels choose their vector form by finer alignment themselves)
bool off_element(const void* p, int dtype) {
  return (reinterpret_cast<uintptr_t>(p) & static_cast<uintptr_t>(element_size(dtype) - 1)) != 0;
}
bool off_vector(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) != 0; }
bool off_word(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3u) != 0; }

// a bf16 / fp32 tensor or its checkpoint: exactly one of the two
int check_kept(const char* what, const void* x, const uint8_t* codes, const uint8_t* scales) {
  if ((codes == nullptr) != (scales == nullptr)) return fail(FFB_ERR_ARG, "%s: codes and scales go together", what);
  if ((x == nullptr) == (codes == nullptr)) return fail(FFB_ERR_ARG, "%s: the tensor or its checkpoint, one of them", what);
  return FFB_OK;
}

// a weight gradient past what the kernels count (rows as TMA coordinates, tiles in 32 bits)
bool wide_grad(int64_t rows, int n, int k) { return rows >= (int64_t(1) << 31) - 4096 || n > (1 << 20) || k > (1 << 20); }

cudaStream_t as_stream(void* s) { return static_cast<cudaStream_t>(s); }

}  // namespace

extern "C" {

int ffb_layernorm_train_fwd(const void* x, void* y, const float* gamma, const float* beta, float* mean, float* rstd,
                            uint8_t* codes, uint8_t* scales, int64_t rows, int c, float eps, int dtype, void* stream) {
  int st = check_rows("layernorm_train_fwd", rows, c, dtype);
  if (st != FFB_OK) return st;
  if (c > kMaxNormChannels)
    return fail(FFB_ERR_UNSUPPORTED, "layernorm_train_fwd: %d channels (at most %d)", c, kMaxNormChannels);
  if (rows == 0) return FFB_OK;
  if (!x || !y || !mean || !rstd) return fail(FFB_ERR_ARG, "layernorm_train_fwd: null pointer");
  if ((codes == nullptr) != (scales == nullptr))
    return fail(FFB_ERR_ARG, "layernorm_train_fwd: codes and scales go together");
  if (x == y) return fail(FFB_ERR_ARG, "layernorm_train_fwd: y must not alias x");
  if (off_vector(x) || off_vector(y) || off_vector(codes) || off_vector(gamma) || off_vector(beta) || off_word(mean) || off_word(rstd))
    return fail(FFB_ERR_ARG, "layernorm_train_fwd: misaligned pointer");
  DeviceInfo info;
  st = device_info(&info);
  if (st != FFB_OK) return st;
  const LayerNormTrain p{x, y, gamma, beta, mean, rstd, codes, scales, rows, c, eps};
  return cuda_status(launch_ln_train(p, dtype == FFB_F32, info.err, as_stream(stream)), "layernorm_train_fwd launch");
}

size_t ffb_layernorm_bwd_workspace_bytes(int64_t rows, int c, int dtype) {
  if (rows <= 0 || c <= 0 || c > kMaxNormChannels) return 0;
  return ln_bwd_workspace_bytes(rows, c, dtype == FFB_F32);
}

int ffb_layernorm_bwd(const void* dy, const void* x, const uint8_t* codes, const uint8_t* scales, const float* mean,
                      const float* rstd, const float* gamma, const void* residual, void* dx, float* dgamma,
                      float* dbeta, void* workspace, size_t workspace_bytes, int64_t rows, int c, int dtype,
                      void* stream) {
  int st = check_rows("layernorm_bwd", rows, c, dtype);
  if (st != FFB_OK) return st;
  if (c > kMaxNormChannels) return fail(FFB_ERR_UNSUPPORTED, "layernorm_bwd: %d channels (at most %d)", c, kMaxNormChannels);
  if (off_word(dgamma) || off_word(dbeta)) return fail(FFB_ERR_ARG, "layernorm_bwd: misaligned pointer");
  DeviceInfo info;
  if (rows == 0) {
    st = device_info(&info);
    if (st != FFB_OK) return st;
    cudaError_t e = cudaSuccess;
    if (dgamma) e = cudaMemsetAsync(dgamma, 0, sizeof(float) * c, as_stream(stream));
    if (dbeta && e == cudaSuccess) e = cudaMemsetAsync(dbeta, 0, sizeof(float) * c, as_stream(stream));
    return cuda_status(static_cast<int>(e), "layernorm_bwd: zero gradients");
  }
  st = check_kept("layernorm_bwd", x, codes, scales);
  if (st != FFB_OK) return st;
  if (!dy || !mean || !rstd || !dx) return fail(FFB_ERR_ARG, "layernorm_bwd: null pointer");
  if (dx == dy || dx == x || dx == residual) return fail(FFB_ERR_ARG, "layernorm_bwd: dx must not alias an input");
  if (off_vector(dy) || off_vector(x) || off_vector(codes) || off_vector(residual) || off_vector(dx) || off_vector(gamma) ||
      off_word(mean) || off_word(rstd))
    return fail(FFB_ERR_ARG, "layernorm_bwd: misaligned pointer");
  if (dgamma || dbeta) {
    const size_t need = ln_bwd_workspace_bytes(rows, c, dtype == FFB_F32);
    if (need > 0 && (!workspace || workspace_bytes < need))
      return fail(FFB_ERR_ARG, "layernorm_bwd: workspace %zu < %zu bytes", workspace ? workspace_bytes : 0, need);
    if ((reinterpret_cast<uintptr_t>(workspace) & 15u) != 0) return fail(FFB_ERR_ARG, "layernorm_bwd: misaligned workspace");
  }
  st = device_info(&info);
  if (st != FFB_OK) return st;
  const LayerNormBwd p{dy, x, codes, scales, mean, rstd, gamma, residual, dx, dgamma, dbeta, workspace, rows, c};
  return cuda_status(launch_ln_bwd(p, dtype == FFB_F32, info.err, as_stream(stream)), "layernorm_bwd launch");
}

int ffb_checkpoint_pack(const void* x, uint8_t* codes, uint8_t* scales, int64_t rows, int c, int dtype, void* stream) {
  int st = check_rows("checkpoint_pack", rows, c, dtype);
  if (st != FFB_OK) return st;
  if (rows == 0) return FFB_OK;
  if (!x || !codes || !scales) return fail(FFB_ERR_ARG, "checkpoint_pack: null pointer");
  if (off_element(x, dtype)) return fail(FFB_ERR_ARG, "checkpoint_pack: misaligned pointer");
  DeviceInfo info;
  st = device_info(&info);
  if (st != FFB_OK) return st;
  return cuda_status(launch_checkpoint_pack(x, codes, scales, rows, c, dtype == FFB_F32, as_stream(stream)),
                     "checkpoint_pack launch");
}

int ffb_checkpoint_unpack(const uint8_t* codes, const uint8_t* scales, void* x, int64_t rows, int c, int dtype,
                          void* stream) {
  int st = check_rows("checkpoint_unpack", rows, c, dtype);
  if (st != FFB_OK) return st;
  if (rows == 0) return FFB_OK;
  if (!x || !codes || !scales) return fail(FFB_ERR_ARG, "checkpoint_unpack: null pointer");
  if (off_element(x, dtype)) return fail(FFB_ERR_ARG, "checkpoint_unpack: misaligned pointer");
  DeviceInfo info;
  st = device_info(&info);
  if (st != FFB_OK) return st;
  return cuda_status(launch_checkpoint_unpack(codes, scales, x, rows, c, dtype == FFB_F32, as_stream(stream)),
                     "checkpoint_unpack launch");
}

size_t ffb_weight_grad_workspace_bytes(int64_t rows, int n, int k, int checkpoint) {
  if (rows <= 0 || n <= 0 || k <= 0 || wide_grad(rows, n, k)) return 0;
  return weight_grad_workspace_bytes(rows, n, k, checkpoint != 0);
}

int ffb_weight_grad(const void* dy, const void* x, const uint8_t* codes, const uint8_t* scales, float* dw,
                    void* workspace, size_t workspace_bytes, int64_t rows, int n, int k, void* stream) {
  if (rows < 0 || n <= 0 || k <= 0)
    return fail(FFB_ERR_ARG, "weight_grad: rows=%lld n=%d k=%d", (long long)rows, n, k);
  if (wide_grad(rows, n, k))
    return fail(FFB_ERR_UNSUPPORTED, "weight_grad: rows=%lld n=%d k=%d", (long long)rows, n, k);
  if (!dw) return fail(FFB_ERR_ARG, "weight_grad: null pointer");
  if (off_word(dw)) return fail(FFB_ERR_ARG, "weight_grad: misaligned pointer");
  DeviceInfo info;
  int st;
  if (rows == 0) {
    st = device_info(&info);
    if (st != FFB_OK) return st;
    return cuda_status(static_cast<int>(cudaMemsetAsync(dw, 0, sizeof(float) * n * static_cast<size_t>(k), as_stream(stream))),
                       "weight_grad: zero gradient");
  }
  st = check_kept("weight_grad", x, codes, scales);
  if (st != FFB_OK) return st;
  if (!dy) return fail(FFB_ERR_ARG, "weight_grad: null pointer");
  if (off_vector(dy) || off_vector(x) || off_vector(codes)) return fail(FFB_ERR_ARG, "weight_grad: misaligned pointer");
  const size_t need = weight_grad_workspace_bytes(rows, n, k, codes != nullptr);
  if (need > 0 && (!workspace || workspace_bytes < need))
    return fail(FFB_ERR_ARG, "weight_grad: workspace %zu < %zu bytes", workspace ? workspace_bytes : 0, need);
  if (off_vector(workspace)) return fail(FFB_ERR_ARG, "weight_grad: misaligned workspace");
  st = device_info(&info);
  if (st != FFB_OK) return st;
  return weight_grad_forward(dy, x, codes, scales, dw, workspace, rows, n, k, info, as_stream(stream));
}

int ffb_swiglu_train_fwd(const void* ab, void* out, uint8_t* codes, uint8_t* scales, int64_t rows, int h, int dtype,
                         void* stream) {
  int st = check_rows("swiglu_train_fwd", rows, 2 * static_cast<int64_t>(h), dtype);
  if (st != FFB_OK) return st;
  if (rows == 0) return FFB_OK;
  if (!ab || !out) return fail(FFB_ERR_ARG, "swiglu_train_fwd: null pointer");
  if ((codes == nullptr) != (scales == nullptr)) return fail(FFB_ERR_ARG, "swiglu_train_fwd: codes and scales go together");
  if (ab == out) return fail(FFB_ERR_ARG, "swiglu_train_fwd: out must not alias ab");
  if (off_element(ab, dtype) || off_element(out, dtype)) return fail(FFB_ERR_ARG, "swiglu_train_fwd: misaligned pointer");
  DeviceInfo info;
  st = device_info(&info);
  if (st != FFB_OK) return st;
  return cuda_status(launch_swiglu_train(ab, out, codes, scales, rows, h, dtype == FFB_F32, as_stream(stream)),
                     "swiglu_train_fwd launch");
}

int ffb_swiglu_bwd(const void* dh, const void* ab, const uint8_t* codes, const uint8_t* scales, void* dab, void* out,
                   int64_t rows, int h, int dtype, void* stream) {
  int st = check_rows("swiglu_bwd", rows, 2 * static_cast<int64_t>(h), dtype);
  if (st != FFB_OK) return st;
  if (rows == 0) return FFB_OK;
  st = check_kept("swiglu_bwd", ab, codes, scales);
  if (st != FFB_OK) return st;
  if (!dh || !dab) return fail(FFB_ERR_ARG, "swiglu_bwd: null pointer");
  if (dab == ab || dab == dh || out == dh || (out != nullptr && (out == ab || out == dab)))
    return fail(FFB_ERR_ARG, "swiglu_bwd: an output must not alias another tensor");
  if (off_element(dh, dtype) || off_element(ab, dtype) || off_element(dab, dtype) || off_element(out, dtype))
    return fail(FFB_ERR_ARG, "swiglu_bwd: misaligned pointer");
  DeviceInfo info;
  st = device_info(&info);
  if (st != FFB_OK) return st;
  return cuda_status(launch_swiglu_bwd(dh, ab, codes, scales, dab, out, rows, h, dtype == FFB_F32, as_stream(stream)),
                     "swiglu_bwd launch");
}

}  // extern "C"
