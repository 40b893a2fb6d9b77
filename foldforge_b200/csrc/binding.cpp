// The torch-facing calls of the training operators and of those around an attention: argument checks,
// outputs, workspaces, device and stream, then one call of the C ABI (include/foldforge_b200.h). A call of
// one token's row costs what the host needs to issue it: about 14 us by ctypes from Python, 7 us from here.
//
// The entry points come in as addresses (bind()), so this module does not link the kernels' library.
// Refusals and errors raise the exceptions of foldforge_b200._lib.
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/extension.h>

#include <optional>
#include <string>

#include "../../include/foldforge_b200.h"

namespace {

namespace py = pybind11;
using at::Tensor;
using OptTensor = std::optional<Tensor>;

constexpr int64_t kBlock = 32;  // channels of a checkpoint that share a scale
constexpr int64_t kMostChannels = int64_t(1) << 30;
// of a weight gradient
constexpr int64_t kMostGradRows = (int64_t(1) << 31) - 4096 - 1, kMostGradChannels = int64_t(1) << 20;

struct Entries {
  decltype(&ffb_last_error) last_error;
  decltype(&ffb_layernorm_train_fwd) layernorm_train_fwd;
  decltype(&ffb_layernorm_bwd_workspace_bytes) layernorm_bwd_workspace_bytes;
  decltype(&ffb_layernorm_bwd) layernorm_bwd;
  decltype(&ffb_checkpoint_pack) checkpoint_pack;
  decltype(&ffb_checkpoint_unpack) checkpoint_unpack;
  decltype(&ffb_weight_grad_workspace_bytes) weight_grad_workspace_bytes;
  decltype(&ffb_weight_grad) weight_grad;
  decltype(&ffb_swiglu_train_fwd) swiglu_train_fwd;
  decltype(&ffb_swiglu_bwd) swiglu_bwd;
  decltype(&ffb_rotary_fwd) rotary_fwd;
  decltype(&ffb_qk_norm_rotary_fwd) qk_norm_rotary_fwd;
  decltype(&ffb_qk_norm_rotary_bwd_workspace_bytes) qk_norm_rotary_bwd_workspace_bytes;
  decltype(&ffb_qk_norm_rotary_bwd) qk_norm_rotary_bwd;
  decltype(&ffb_dropout) dropout;
} entries;

[[noreturn]] void raise(const char* name, int status, const std::string& message) {
  const py::module_ lib = py::module_::import("foldforge_b200._lib");
  const py::object type = lib.attr(status == FFB_ERR_UNSUPPORTED ? "UnsupportedCall" : "KernelError");
  const py::object error = type(name, status, message);
  PyErr_SetObject(type.ptr(), error.ptr());
  throw py::error_already_set();
}
[[noreturn]] void refuse(const char* name, const std::string& message) { raise(name, FFB_ERR_UNSUPPORTED, message); }

void check(const char* name, int status) {
  if (status != FFB_OK) raise(name, status, entries.last_error());
}

std::string text(c10::IntArrayRef shape) {
  std::string s = "[";
  for (size_t i = 0; i < shape.size(); ++i) s += (i ? ", " : "") + std::to_string(shape[i]);
  return s + "]";
}
std::string text(const Tensor& t) { return std::string(c10::toString(t.scalar_type())) + " " + text(t.sizes()) + " on " + t.device().str(); }

int dtype_of(at::ScalarType t) { return t == at::kFloat ? FFB_F32 : FFB_BF16; }

// Outside autograd and dense. (Called under a guard that records nothing.)
Tensor dense(const Tensor& t) { return t.is_contiguous() ? t : t.contiguous(); }

// a copy of a view that does not start on a 16-byte boundary
Tensor aligned(const Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 ? t : t.clone(); }

// The entry points take channels as an int: wider rows are refused before they are narrowed.
void check_channels(const char* name, c10::IntArrayRef shape) {
  if (shape.back() < 0 || shape.back() > kMostChannels) refuse(name, std::to_string(shape.back()) + " channels");
}

// The first tensor of a call: bf16 (or fp32) rows of at least one channel.
void check_rows(const char* name, const Tensor& x, bool fp32 = true) {
  if (x.scalar_type() != at::kBFloat16 && !(fp32 && x.scalar_type() == at::kFloat))
    refuse(name, std::string("dtype ") + c10::toString(x.scalar_type()) + (fp32 ? " (takes bf16 or fp32)" : " (takes bf16)"));
  if (x.dim() == 0 || x.size(-1) == 0) refuse(name, "shape " + text(x.sizes()) + " has no channels");
  check_channels(name, x.sizes());
}
Tensor rows_of(const char* name, const Tensor& x) {
  check_rows(name, x);
  return dense(x);
}

// Checks of shapes come before this one, so that they can be tested anywhere.
void need_cuda(const char* name, const Tensor& x) {
  if (!x.is_cuda()) refuse(name, "tensor is not on a CUDA device");
}

Tensor beside(const char* name, const char* what, const Tensor& x, const Tensor& t, c10::IntArrayRef shape, at::ScalarType dtype) {
  if (t.sizes() != shape || t.scalar_type() != dtype || t.device() != x.device())
    refuse(name, std::string(what) + " is " + text(t) + ", not " + c10::toString(dtype) + " " + text(shape) + " on " + x.device().str());
  return dense(t);
}

// a norm's weight or bias in fp32
Tensor vector(const char* name, const char* what, const Tensor& x, const Tensor& t) {
  if (t.dim() != 1 || t.size(0) != x.size(-1) || t.device() != x.device() || !t.is_floating_point())
    refuse(name, std::string(what) + " is " + text(t) + ", beside " + text(x));
  return aligned(t.scalar_type() == at::kFloat ? dense(t) : t.to(at::kFloat).contiguous());
}

// New tensors on x's CUDA device, from the allocator without the dispatcher (a call of a token's q and k makes two, its
// backward pass five)
Tensor made(const Tensor& x, c10::IntArrayRef shape, at::ScalarType dtype) {
  return Tensor(at::detail::empty_cuda(shape, dtype, x.device(), std::nullopt));
}
Tensor bytes(const Tensor& x, int64_t n) { return made(x, {n}, at::kByte); }
Tensor floats(const Tensor& x, c10::IntArrayRef shape) { return made(x, shape, at::kFloat); }
Tensor like(const Tensor& x, c10::IntArrayRef shape) { return made(x, shape, x.scalar_type()); }

// ---- checkpoints: codes, then (from the next multiple of 16 bytes on) scales
int64_t scales_at(int64_t codes) { return (codes + 15) / 16 * 16; }
int64_t checkpoint_bytes(int64_t codes, int64_t c) { return scales_at(codes) + codes / c * ((c + kBlock - 1) / kBlock); }

// What a backward pass reads: a tensor, or a checkpoint's bytes with the shape and dtype it stands for.
struct Kept {
  Tensor tensor;
  const void* x = nullptr;
  const uint8_t* codes = nullptr;
  const uint8_t* scales = nullptr;
};
Kept kept_of(const char* name, const Tensor& x, const Tensor& t, bool checkpoint, c10::IntArrayRef shape, at::ScalarType dtype) {
  Kept k;
  if (!checkpoint) {
    k.tensor = beside(name, "the kept activation", x, t, shape, dtype);
    k.x = k.tensor.data_ptr();
    return k;
  }
  const int64_t codes = c10::multiply_integers(shape);
  k.tensor = beside(name, "the checkpoint", x, t, {checkpoint_bytes(codes, shape.back())}, at::kByte);
  k.codes = static_cast<const uint8_t*>(k.tensor.data_ptr());
  k.scales = k.codes + scales_at(codes);
  return k;
}

// The device of a call's tensors, its current stream, and no autograd while it runs.
struct Call {
  c10::cuda::CUDAGuard device;
  void* stream;
  explicit Call(const Tensor& x) : device(x.device()), stream(c10::cuda::getCurrentCUDAStream(x.device().index()).stream()) {}
};

float* pointer(const OptTensor& t) { return t ? t->data_ptr<float>() : nullptr; }

Tensor checkpoint_pack(const Tensor& x_in) {
  at::NoGradGuard no_grad;
  const char* name = "checkpoint_pack";
  const Tensor x = rows_of(name, x_in);
  need_cuda(name, x);
  Call call(x);
  const int64_t n = x.numel(), c = x.size(-1);
  const Tensor data = bytes(x, checkpoint_bytes(n, c));
  uint8_t* codes = data.data_ptr<uint8_t>();
  check(name, entries.checkpoint_pack(x.data_ptr(), codes, codes + scales_at(n), n / c, static_cast<int>(c), dtype_of(x.scalar_type()), call.stream));
  return data;
}

Tensor checkpoint_unpack(const Tensor& data_in, const std::vector<int64_t>& shape, at::ScalarType dtype) {
  at::NoGradGuard no_grad;
  const char* name = "checkpoint_unpack";
  if ((dtype != at::kBFloat16 && dtype != at::kFloat) || shape.empty() || shape.back() == 0)
    refuse(name, std::string("of a ") + c10::toString(dtype) + " " + text(shape) + " activation");
  check_channels(name, shape);
  const Kept k = kept_of(name, data_in, data_in, true, shape, dtype);
  need_cuda(name, data_in);
  Call call(data_in);
  const Tensor x = made(data_in, shape, dtype);
  const int64_t c = shape.back();
  check(name, entries.checkpoint_unpack(k.codes, k.scales, x.data_ptr(), x.numel() / c, static_cast<int>(c), dtype_of(dtype), call.stream));
  return x;
}

std::tuple<Tensor, Tensor, Tensor> layer_norm_train(const Tensor& x_in, const OptTensor& weight, const OptTensor& bias, double eps,
                                                    bool checkpoint) {
  at::NoGradGuard no_grad;
  const char* name = "layer_norm_train";
  const Tensor x = aligned(rows_of(name, x_in));
  OptTensor w, b;
  if (weight) w = vector(name, "weight", x, *weight);
  if (bias) b = vector(name, "bias", x, *bias);
  need_cuda(name, x);
  Call call(x);
  const int64_t n = x.numel(), c = x.size(-1), rows = n / c;
  const Tensor y = like(x, x.sizes()), stats = floats(x, {2, rows});
  float* mean = stats.data_ptr<float>();
  Tensor kept = x.requires_grad() ? x.detach() : x;
  uint8_t* codes = nullptr;
  if (checkpoint) {
    kept = bytes(x, checkpoint_bytes(n, c));
    codes = kept.data_ptr<uint8_t>();
  }
  check(name, entries.layernorm_train_fwd(x.data_ptr(), y.data_ptr(), pointer(w), pointer(b), mean, mean + rows, codes,
                                          codes ? codes + scales_at(n) : nullptr, rows, static_cast<int>(c), static_cast<float>(eps),
                                          dtype_of(x.scalar_type()), call.stream));
  return {y, kept, stats};
}

std::tuple<Tensor, OptTensor, OptTensor> layer_norm_backward(const Tensor& dy_in, const Tensor& kept, bool checkpoint, const Tensor& stats_in,
                                                             const OptTensor& weight, bool weight_gradient, bool bias,
                                                             const OptTensor& residual_in) {
  at::NoGradGuard no_grad;
  const char* name = "layer_norm_backward";
  const Tensor dy = aligned(rows_of(name, dy_in));
  const int64_t c = dy.size(-1), rows = dy.numel() / c;
  kept_of(name, dy, kept, checkpoint, dy.sizes(), dy.scalar_type());
  const Kept k = kept_of(name, dy, aligned(dense(kept)), checkpoint, dy.sizes(), dy.scalar_type());
  const Tensor stats = beside(name, "stats", dy, stats_in, {2, rows}, at::kFloat);
  OptTensor w, residual, dweight, dbias, ws;
  if (weight) w = vector(name, "weight", dy, *weight);
  if (residual_in) residual = aligned(beside(name, "residual", dy, *residual_in, dy.sizes(), dy.scalar_type()));
  need_cuda(name, dy);
  Call call(dy);
  const Tensor dx = like(dy, dy.sizes());
  if (w && weight_gradient) dweight = floats(dy, {c});
  if (bias) dbias = floats(dy, {c});
  const int dtype = dtype_of(dy.scalar_type());
  const size_t size = dweight || dbias ? entries.layernorm_bwd_workspace_bytes(rows, static_cast<int>(c), dtype) : 0;
  if (size) ws = bytes(dy, static_cast<int64_t>(size));
  const float* mean = stats.data_ptr<float>();
  check(name, entries.layernorm_bwd(dy.data_ptr(), k.x, k.codes, k.scales, mean, mean + rows, pointer(w),
                                    residual ? residual->data_ptr() : nullptr, dx.data_ptr(), pointer(dweight), pointer(dbias),
                                    ws ? ws->data_ptr() : nullptr, size, rows, static_cast<int>(c), dtype, call.stream));
  return {dx, dweight, dbias};
}

Tensor weight_grad(const Tensor& dy_in, const Tensor& kept, bool checkpoint, const std::vector<int64_t>& shape, at::ScalarType dtype) {
  at::NoGradGuard no_grad;
  const char* name = "weight_grad";
  check_rows(name, dy_in, false);
  if (shape.empty() || shape.back() <= 0 || c10::IntArrayRef(shape).slice(0, shape.size() - 1) != dy_in.sizes().slice(0, dy_in.dim() - 1))
    refuse(name, "rows of dy " + text(dy_in.sizes()) + " and x " + text(shape));
  if (dtype != at::kBFloat16) refuse(name, std::string("x is ") + c10::toString(dtype) + " (takes bf16)");
  const int64_t n = dy_in.size(-1), k = shape.back(), rows = dy_in.numel() / n;
  if (rows > kMostGradRows || n > kMostGradChannels || k > kMostGradChannels)
    refuse(name, std::to_string(rows) + " rows of " + std::to_string(n) + " and " + std::to_string(k) + " channels");
  Tensor dy = dense(dy_in);
  kept_of(name, dy, kept, checkpoint, shape, dtype);
  need_cuda(name, dy);
  Call call(dy);
  dy = aligned(dy);
  const Kept x = kept_of(name, dy, aligned(dense(kept)), checkpoint, shape, dtype);
  const Tensor dw = floats(dy, {n, k});
  const size_t size = entries.weight_grad_workspace_bytes(rows, static_cast<int>(n), static_cast<int>(k), checkpoint);
  OptTensor ws;
  if (size) ws = bytes(dy, static_cast<int64_t>(size));
  check(name, entries.weight_grad(dy.data_ptr(), x.x, x.codes, x.scales, dw.data_ptr<float>(), ws ? ws->data_ptr() : nullptr, size, rows,
                                  static_cast<int>(n), static_cast<int>(k), call.stream));
  return dw;
}

std::tuple<Tensor, Tensor> swiglu_train(const Tensor& ab_in, bool checkpoint) {
  at::NoGradGuard no_grad;
  const char* name = "swiglu_train";
  const Tensor ab = rows_of(name, ab_in);
  const int64_t n = ab.numel(), c = ab.size(-1);
  if (c % 2) refuse(name, std::to_string(c) + " channels are not [a | b]");
  need_cuda(name, ab);
  Call call(ab);
  auto shape = ab.sizes().vec();
  shape.back() = c / 2;
  const Tensor out = like(ab, shape);
  Tensor kept = ab.requires_grad() ? ab.detach() : ab;
  uint8_t* codes = nullptr;
  if (checkpoint) {
    kept = bytes(ab, checkpoint_bytes(n, c));
    codes = kept.data_ptr<uint8_t>();
  }
  check(name, entries.swiglu_train_fwd(ab.data_ptr(), out.data_ptr(), codes, codes ? codes + scales_at(n) : nullptr, n / c,
                                       static_cast<int>(c / 2), dtype_of(ab.scalar_type()), call.stream));
  return {out, kept};
}

std::tuple<Tensor, OptTensor> swiglu_backward(const Tensor& dh_in, const Tensor& kept, bool checkpoint, bool output) {
  at::NoGradGuard no_grad;
  const char* name = "swiglu_backward";
  const Tensor dh = rows_of(name, dh_in);
  const int64_t h = dh.size(-1);
  auto shape = dh.sizes().vec();
  shape.back() = 2 * h;
  const Kept k = kept_of(name, dh, kept, checkpoint, shape, dh.scalar_type());
  need_cuda(name, dh);
  Call call(dh);
  const Tensor dab = like(dh, shape);
  OptTensor out;
  if (output) out = like(dh, dh.sizes());
  check(name, entries.swiglu_bwd(dh.data_ptr(), k.x, k.codes, k.scales, dab.data_ptr(), out ? out->data_ptr() : nullptr, dh.numel() / h,
                                 static_cast<int>(h), dtype_of(dh.scalar_type()), call.stream));
  return {dab, out};
}

// ---- around an attention: heads [tokens, heads, channels] or [batch, tokens, heads, channels] as they lie
constexpr int64_t kMostHeadChannels = 512;

struct Heads {
  Tensor t;
  ffb_heads view{};
  const ffb_heads* at() const { return t.defined() ? &view : nullptr; }
};

// `like`: the tensor whose dtype, device and (but for the heads, where `heads`) shape this one has; an output's
// channels have to be dense as they lie.
Heads heads_of(const char* name, const char* what, const Tensor& t_in, const Tensor& like, bool heads, bool output = false) {
  const int64_t dim = like.dim();
  bool same = t_in.dim() == dim && t_in.scalar_type() == like.scalar_type() && t_in.device() == like.device();
  for (int64_t i = 0; same && i < dim; ++i) same = t_in.size(i) == like.size(i) || (heads && i == dim - 2);
  if (!same) refuse(name, std::string(what) + " is " + text(t_in) + ", beside " + text(like));
  Heads h;
  const bool dense_rows = t_in.stride(-1) == 1 || t_in.size(-1) <= 1;
  if (output && !dense_rows) refuse(name, std::string(what) + "'s channels are " + std::to_string(t_in.stride(-1)) + " elements apart");
  h.t = dense_rows ? t_in : t_in.contiguous();
  h.view = {h.t.data_ptr(), dim == 4 ? h.t.stride(0) : 0, h.t.stride(dim - 3), h.t.stride(dim - 2), h.t.size(dim - 2)};
  return h;
}

// q, the first tensor of a call
Heads first_heads(const char* name, const Tensor& q) {
  if (q.scalar_type() != at::kBFloat16 && q.scalar_type() != at::kFloat)
    refuse(name, std::string("dtype ") + c10::toString(q.scalar_type()) + " (takes bf16 or fp32)");
  if (q.dim() != 3 && q.dim() != 4) refuse(name, "shape " + text(q.sizes()) + " is neither [tokens, heads, channels] nor [batch, tokens, heads, channels]");
  if (q.size(-1) < 1 || q.size(-1) > kMostHeadChannels)
    refuse(name, std::to_string(q.size(-1)) + " channels a head (1 to " + std::to_string(kMostHeadChannels) + ")");
  return heads_of(name, "q", q, q, false);
}

Heads output_heads(const char* name, const char* what, const Heads& x, const OptTensor& out) {
  return heads_of(name, what, out ? *out : like(x.t, x.t.sizes()), x.t, false, true);
}

// A tensor of the caller's to write. Nothing here is recorded: one that autograd follows would keep the gradient of what it
// held before. (Called outside the guard.)
void need_unfollowed(const char* name, const char* what, const OptTensor& out) {
  if (out && out->requires_grad() && at::GradMode::is_enabled()) refuse(name, std::string(what) + " to write requires a gradient");
}
// counts it as written, so that a backward pass which kept it (or memory that it shares) refuses to read it
void written(const OptTensor& out) {
  if (out && !out->is_inference()) out->unsafeGetTensorImpl()->bump_version();
}

using Table = std::tuple<Tensor, Tensor, int64_t, bool>;  // quarter turns, the pairs' axes, axes, interleaved

struct Rotary {
  Tensor positions, quarters, axes;
  ffb_rotary params{};
};
Rotary rotary_of(const char* name, const Tensor& q, const OptTensor& positions, const std::optional<Table>& table, bool inverse) {
  Rotary r;
  if (positions.has_value() != table.has_value()) refuse(name, "positions and their table go together");
  if (!table) return r;
  int64_t axes;
  bool interleaved;
  std::tie(r.quarters, r.axes, axes, interleaved) = *table;
  r.positions = *positions;
  const int64_t pairs = r.quarters.numel(), d = r.positions.dim(), qd = q.dim();
  if (r.quarters.dim() != 1 || r.quarters.scalar_type() != at::kDouble || r.axes.sizes() != r.quarters.sizes() ||
      r.axes.scalar_type() != at::kInt || r.quarters.device() != q.device() || r.axes.device() != q.device() ||
      !r.quarters.is_contiguous() || !r.axes.is_contiguous())
    refuse(name, "the table is " + text(r.quarters) + " and " + text(r.axes) + ", beside " + text(q));
  if (pairs > q.size(-1) / 2) refuse(name, std::to_string(pairs) + " pairs of " + std::to_string(q.size(-1)) + " channels");
  const at::ScalarType type = r.positions.scalar_type();
  if (type != at::kInt && type != at::kLong && type != at::kFloat)
    refuse(name, std::string("positions are ") + c10::toString(type) + " (takes int32, int64 or fp32)");
  const int64_t batch = qd == 4 ? q.size(0) : 1;
  if (r.positions.device() != q.device() || d < 2 || d > 3 || r.positions.size(d - 2) != q.size(qd - 3) ||
      (d == 3 && r.positions.size(0) != batch && r.positions.size(0) != 1))
    refuse(name, "positions are " + text(r.positions) + ", beside " + text(q));
  if (axes < 1 || r.positions.size(d - 1) < axes)
    refuse(name, "positions of " + std::to_string(r.positions.size(d - 1)) + " axes for a table of " + std::to_string(axes));
  r.params = {r.positions.data_ptr(), d == 3 && r.positions.size(0) > 1 ? r.positions.stride(0) : 0, r.positions.stride(d - 2),
              r.positions.stride(d - 1), r.quarters.data_ptr<double>(), r.axes.data_ptr<int32_t>(),
              type == at::kInt ? FFB_POSITION_I32 : type == at::kLong ? FFB_POSITION_I64 : FFB_POSITION_F32,
              static_cast<int>(axes), static_cast<int>(pairs), interleaved, inverse};
  return r;
}

int64_t batch_of(const Tensor& q) { return q.dim() == 4 ? q.size(0) : 1; }
int64_t tokens_of(const Tensor& q) { return q.size(-3); }

std::tuple<Tensor, OptTensor> heads_forward(const char* name, bool norm, const Tensor& q_in, const OptTensor& k_in,
                                            const OptTensor& positions, const std::optional<Table>& table, bool inverse,
                                            const OptTensor& q_weight, const OptTensor& k_weight, double eps,
                                            const OptTensor& q_out_in, const OptTensor& k_out_in) {
  need_unfollowed(name, "q's output", q_out_in);
  need_unfollowed(name, "k's output", k_out_in);
  at::NoGradGuard no_grad;
  const Heads q = first_heads(name, q_in);
  Heads k, q_out, k_out;
  if (k_in) k = heads_of(name, "k", *k_in, q_in, true);
  if (!k_in && (k_weight || k_out_in)) refuse(name, "k's weight or output without k");
  const Rotary r = rotary_of(name, q_in, positions, table, inverse);
  OptTensor qw, kw;
  if (q_weight) qw = vector(name, "q's weight", q.t, *q_weight);
  if (k_weight) kw = vector(name, "k's weight", q.t, *k_weight);
  if (q_out_in) output_heads(name, "q's output", q, q_out_in);
  if (k_out_in) output_heads(name, "k's output", k, k_out_in);
  need_cuda(name, q.t);
  Call call(q.t);
  q_out = output_heads(name, "q's output", q, q_out_in);
  if (k_in) k_out = output_heads(name, "k's output", k, k_out_in);
  const int channels = static_cast<int>(q.t.size(-1)), dtype = dtype_of(q.t.scalar_type());
  const int64_t batch = batch_of(q.t), tokens = tokens_of(q.t);
  check(name, norm ? entries.qk_norm_rotary_fwd(q.at(), k.at(), q_out.at(), k_out.at(), pointer(qw), pointer(kw),
                                                static_cast<float>(eps), &r.params, batch, tokens, channels, dtype, call.stream)
                   : entries.rotary_fwd(q.at(), k.at(), q_out.at(), k_out.at(), &r.params, batch, tokens, channels, dtype, call.stream));
  written(q_out_in);
  written(k_out_in);
  return {q_out.t, k_in ? OptTensor(k_out.t) : OptTensor()};
}

std::tuple<Tensor, OptTensor> rotary(const Tensor& q, const OptTensor& k, const Tensor& positions, const Table& table, bool inverse,
                                     const OptTensor& q_out, const OptTensor& k_out) {
  return heads_forward("rotary", false, q, k, positions, table, inverse, {}, {}, 0.0, q_out, k_out);
}

std::tuple<Tensor, OptTensor> qk_norm_rotary(const Tensor& q, const OptTensor& k, const OptTensor& positions,
                                             const std::optional<Table>& table, const OptTensor& q_weight, const OptTensor& k_weight,
                                             double eps, const OptTensor& q_out, const OptTensor& k_out) {
  return heads_forward("qk_norm_rotary", true, q, k, positions, table, false, q_weight, k_weight, eps, q_out, k_out);
}

std::tuple<Tensor, OptTensor, OptTensor, OptTensor> qk_norm_rotary_backward(
    const Tensor& dq_out, const OptTensor& dk_out, const Tensor& q_in, const OptTensor& k_in, const OptTensor& positions,
    const std::optional<Table>& table, const OptTensor& q_weight, const OptTensor& k_weight, double eps, bool weight_gradient,
    const OptTensor& dq_in, const OptTensor& dk_in) {
  const char* name = "qk_norm_rotary_backward";
  need_unfollowed(name, "q's gradient", dq_in);
  need_unfollowed(name, "k's gradient", dk_in);
  at::NoGradGuard no_grad;
  const Heads q = first_heads(name, q_in);
  const Heads dy_q = heads_of(name, "the gradient of q's output", dq_out, q_in, false);
  Heads k, dy_k, dq, dk;
  if (k_in.has_value() != dk_out.has_value()) refuse(name, "k and the gradient of its output go together");
  if (!k_in && (k_weight || dk_in)) refuse(name, "k's weight or gradient without k");
  if (k_in) {
    k = heads_of(name, "k", *k_in, q_in, true);
    dy_k = heads_of(name, "the gradient of k's output", *dk_out, *k_in, false);
  }
  const Rotary r = rotary_of(name, q_in, positions, table, false);
  OptTensor qw, kw, dqw, dkw, ws;
  if (q_weight) qw = vector(name, "q's weight", q.t, *q_weight);
  if (k_weight) kw = vector(name, "k's weight", q.t, *k_weight);
  if (dq_in) output_heads(name, "q's gradient", q, dq_in);
  if (dk_in) output_heads(name, "k's gradient", k, dk_in);
  need_cuda(name, q.t);
  Call call(q.t);
  dq = output_heads(name, "q's gradient", q, dq_in);
  if (k_in) dk = output_heads(name, "k's gradient", k, dk_in);
  const int64_t batch = batch_of(q.t), tokens = tokens_of(q.t), c = q.t.size(-1);
  const int channels = static_cast<int>(c), dtype = dtype_of(q.t.scalar_type());
  size_t size = 0;
  if (weight_gradient && (qw || kw)) {
    if (qw) dqw = floats(q.t, {c});
    if (kw) dkw = floats(q.t, {c});
    size = entries.qk_norm_rotary_bwd_workspace_bytes(batch, tokens, q.view.heads, k_in ? k.view.heads : 0, channels, dtype);
    if (size) ws = bytes(q.t, static_cast<int64_t>(size));
  }
  check(name, entries.qk_norm_rotary_bwd(dy_q.at(), dy_k.at(), q.at(), k.at(), dq.at(), dk.at(), pointer(qw), pointer(kw), pointer(dqw),
                                         pointer(dkw), static_cast<float>(eps), &r.params, ws ? ws->data_ptr() : nullptr, size, batch,
                                         tokens, channels, dtype, call.stream));
  written(dq_in);
  written(dk_in);
  return {dq.t, k_in ? OptTensor(dk.t) : OptTensor(), dqw, dkw};
}

// x dropped and scaled (plus the residual) in out_dtype; axes: those whose positions share a mask, ascending
Tensor dropout(const char* name, const Tensor& x_in, double p, uint64_t seed, uint64_t offset, const OptTensor& device_seed,
               const OptTensor& residual_in, const std::vector<int64_t>& axes, at::ScalarType out_dtype) {
  at::NoGradGuard no_grad;
  for (const at::ScalarType t : {x_in.scalar_type(), out_dtype})
    if (t != at::kBFloat16 && t != at::kFloat) refuse(name, std::string("dtype ") + c10::toString(t) + " (takes bf16 or fp32)");
  if (!(p >= 0.0 && p <= 1.0)) refuse(name, "p = " + std::to_string(p));
  int64_t outer = 1, shared = 1, inner = 1;
  if (axes.empty()) {
    inner = x_in.numel();
  } else {
    for (size_t i = 0; i < axes.size(); ++i)
      if (axes[i] < 0 || axes[i] >= x_in.dim() || axes[i] != axes[0] + static_cast<int64_t>(i))
        refuse(name, "shared axes " + text(axes) + " of " + text(x_in.sizes()) + " (axes beside one another)");
    for (int64_t i = 0; i < x_in.dim(); ++i) (i < axes.front() ? outer : i > axes.back() ? inner : shared) *= x_in.size(i);
  }
  OptTensor residual;
  if (residual_in) residual = beside(name, "residual", x_in, *residual_in, x_in.sizes(), out_dtype);
  if (device_seed && (device_seed->scalar_type() != at::kLong || device_seed->dim() != 1 || device_seed->size(0) != 2 ||
                      !device_seed->is_contiguous() || device_seed->device() != x_in.device()))
    refuse(name, "seed is " + text(*device_seed) + ", not Long [2] on " + x_in.device().str());
  need_cuda(name, x_in);
  Call call(x_in);
  const Tensor x = dense(x_in);
  const Tensor out = made(x, x.sizes(), out_dtype);
  check(name, entries.dropout(x.data_ptr(), dtype_of(x.scalar_type()), residual ? residual->data_ptr() : nullptr, out.data_ptr(),
                              dtype_of(out_dtype), outer, shared, inner, p, seed, offset,
                              device_seed ? reinterpret_cast<const uint64_t*>(device_seed->data_ptr<int64_t>()) : nullptr, call.stream));
  return out;
}

template <typename F>
void take(const py::dict& addresses, const char* name, F& f) {
  f = reinterpret_cast<F>(addresses[name].cast<uintptr_t>());
}

}  // namespace

PYBIND11_MODULE(_binding, m) {
  m.def("bind", [](const py::dict& a) {
    take(a, "ffb_last_error", entries.last_error);
    take(a, "ffb_layernorm_train_fwd", entries.layernorm_train_fwd);
    take(a, "ffb_layernorm_bwd_workspace_bytes", entries.layernorm_bwd_workspace_bytes);
    take(a, "ffb_layernorm_bwd", entries.layernorm_bwd);
    take(a, "ffb_checkpoint_pack", entries.checkpoint_pack);
    take(a, "ffb_checkpoint_unpack", entries.checkpoint_unpack);
    take(a, "ffb_weight_grad_workspace_bytes", entries.weight_grad_workspace_bytes);
    take(a, "ffb_weight_grad", entries.weight_grad);
    take(a, "ffb_swiglu_train_fwd", entries.swiglu_train_fwd);
    take(a, "ffb_swiglu_bwd", entries.swiglu_bwd);
    take(a, "ffb_rotary_fwd", entries.rotary_fwd);
    take(a, "ffb_qk_norm_rotary_fwd", entries.qk_norm_rotary_fwd);
    take(a, "ffb_qk_norm_rotary_bwd_workspace_bytes", entries.qk_norm_rotary_bwd_workspace_bytes);
    take(a, "ffb_qk_norm_rotary_bwd", entries.qk_norm_rotary_bwd);
    take(a, "ffb_dropout", entries.dropout);
  });
  m.def("checkpoint_pack", &checkpoint_pack);
  m.def("checkpoint_unpack", &checkpoint_unpack);
  m.def("layer_norm_train", &layer_norm_train);
  m.def("layer_norm_backward", &layer_norm_backward);
  m.def("weight_grad", &weight_grad);
  m.def("swiglu_train", &swiglu_train);
  m.def("swiglu_backward", &swiglu_backward);
  m.def("rotary", &rotary);
  m.def("qk_norm_rotary", &qk_norm_rotary);
  m.def("qk_norm_rotary_backward", &qk_norm_rotary_backward);
  m.def("dropout", &dropout);
}
