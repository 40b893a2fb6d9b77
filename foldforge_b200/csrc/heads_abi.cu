// The C ABI of the norm and rotation of queries and keys: argument checks around heads.cu.
#include <math.h>

#include "../../include/foldforge_b200.h"
#include "abi_util.h"
#include "kernels.h"

using namespace ffb;

namespace {

constexpr int64_t kMostElements = int64_t(1) << 46;  // that any tensor spans

cudaStream_t as_stream(void* s) { return static_cast<cudaStream_t>(s); }

struct Sizes {
  const char* what;
  int64_t batch, tokens;
  int channels, element;  // bytes of an element
};

int check_sizes(Sizes* s, const char* what, int64_t batch, int64_t tokens, int channels, int dtype) {
  if (batch < 0 || tokens < 0 || channels <= 0)
    return fail(FFB_ERR_ARG, "%s: batch=%lld tokens=%lld channels=%d", what, (long long)batch, (long long)tokens, channels);
  if (channels > kMaxHeadChannels) return fail(FFB_ERR_UNSUPPORTED, "%s: %d channels (at most %d)", what, channels, kMaxHeadChannels);
  const int64_t most = (int64_t(1) << 31) - 2;
  if (batch > most || (batch > 0 && tokens > most / batch)) return fail(FFB_ERR_UNSUPPORTED, "%s: too many tokens", what);
  if (dtype != FFB_BF16 && dtype != FFB_F32) return fail(FFB_ERR_UNSUPPORTED, "%s: dtype %d", what, dtype);
  *s = {what, batch, tokens, channels, dtype == FFB_F32 ? 4 : 2};
  return FFB_OK;
}

bool empty(const Sizes& s, const ffb_heads& h) { return s.batch == 0 || s.tokens == 0 || h.heads == 0; }

// elements from the first to behind the last of a view whose strides are checked
int64_t extent(const Sizes& s, const ffb_heads& h) {
  return (s.batch - 1) * h.batch_stride + (s.tokens - 1) * h.token_stride + (h.heads - 1) * h.head_stride + s.channels;
}

bool stride_ok(int64_t n, int64_t stride) { return stride >= 0 && (n <= 1 || stride <= kMostElements / n); }

int check_view(const Sizes& s, const char* name, const ffb_heads* h, int64_t heads) {
  if (h == nullptr) return fail(FFB_ERR_ARG, "%s: %s is missing", s.what, name);
  if (h->heads != heads) return fail(FFB_ERR_ARG, "%s: %s has %lld heads, not %lld", s.what, name, (long long)h->heads, (long long)heads);
  if (heads < 0) return fail(FFB_ERR_ARG, "%s: %s has %lld heads", s.what, name, (long long)heads);
  if (heads > (1 << 20)) return fail(FFB_ERR_UNSUPPORTED, "%s: %lld heads", s.what, (long long)heads);
  if (empty(s, *h)) return FFB_OK;
  if (h->data == nullptr) return fail(FFB_ERR_ARG, "%s: %s is a null pointer", s.what, name);
  if ((reinterpret_cast<uintptr_t>(h->data) & static_cast<uintptr_t>(s.element - 1)) != 0)
    return fail(FFB_ERR_ARG, "%s: %s is misaligned", s.what, name);
  if (!stride_ok(s.batch, h->batch_stride) || !stride_ok(s.tokens, h->token_stride) || !stride_ok(heads, h->head_stride) ||
      extent(s, *h) > kMostElements)
    return fail(FFB_ERR_ARG, "%s: strides of %s", s.what, name);
  return FFB_OK;
}

// An output's elements are distinct: from the smallest stride up, each axis steps over all that lies below it.
int check_output(const Sizes& s, const char* name, const ffb_heads& h) {
  if (empty(s, h)) return FFB_OK;
  int64_t n[3] = {s.batch, s.tokens, h.heads}, stride[3] = {h.batch_stride, h.token_stride, h.head_stride};
  for (int i = 0; i < 3; ++i)
    for (int j = i + 1; j < 3; ++j)
      if (stride[j] < stride[i]) {
        const int64_t a = stride[i], b = n[i];
        stride[i] = stride[j], n[i] = n[j], stride[j] = a, n[j] = b;
      }
  int64_t span = s.channels;
  for (int i = 0; i < 3; ++i) {
    if (n[i] <= 1) continue;
    if (stride[i] < span) return fail(FFB_ERR_ARG, "%s: elements of %s overlap", s.what, name);
    span += (n[i] - 1) * stride[i];
  }
  return FFB_OK;
}

bool same_view(const Sizes& s, const ffb_heads& a, const ffb_heads& b) {
  return a.data == b.data && a.heads == b.heads && (s.batch == 1 || a.batch_stride == b.batch_stride) &&
         (s.tokens == 1 || a.token_stride == b.token_stride) && (a.heads == 1 || a.head_stride == b.head_stride);
}

// Where b starts behind a, and their sizes and strides on the batch, the tokens and the heads, in elements.
struct Beside {
  int64_t delta, channels, na[3], nb[3], sa[3], sb[3];
};
// Two views share no element over the axes of the set `left`: one ends before the other begins, or an axis that they step
// along alike has steps that reach over both of their parts, and within a step these share none.
bool apart(const Beside& v, unsigned left) {
  int64_t wa = v.channels, wb = v.channels;
  for (int i = 0; i < 3; ++i)
    if (left >> i & 1) {
      wa += (v.na[i] - 1) * v.sa[i];
      wb += (v.nb[i] - 1) * v.sb[i];
    }
  if (wa <= v.delta || wb <= -v.delta) return true;
  for (int i = 0; i < 3; ++i) {
    if (!(left >> i & 1) || (v.na[i] == 1 && v.nb[i] == 1)) continue;
    const int64_t step = v.na[i] > 1 ? v.sa[i] : v.sb[i];
    if (v.na[i] > 1 && v.nb[i] > 1 && v.sb[i] != step) continue;
    const int64_t a_end = wa - (v.na[i] - 1) * v.sa[i], b_end = v.delta + wb - (v.nb[i] - 1) * v.sb[i];
    const int64_t span = (a_end > b_end ? a_end : b_end) - (v.delta < 0 ? v.delta : 0);
    if (span <= step && apart(v, left & ~(1u << i))) return true;
  }
  return false;
}
bool apart(const Sizes& s, const ffb_heads& a, const ffb_heads& b) {
  const int64_t bytes = static_cast<int64_t>(reinterpret_cast<uintptr_t>(b.data)) - static_cast<int64_t>(reinterpret_cast<uintptr_t>(a.data));
  if (bytes % s.element != 0) return false;
  return apart(Beside{bytes / s.element, s.channels, {s.batch, s.tokens, a.heads}, {s.batch, s.tokens, b.heads},
                      {a.batch_stride, a.token_stride, a.head_stride}, {b.batch_stride, b.token_stride, b.head_stride}}, 7u);
}

int check_rotary(const Sizes& s, const ffb_rotary* r) {
  if (r == nullptr) return fail(FFB_ERR_ARG, "%s: no rotary", s.what);
  if (r->pairs < 0 || r->pairs > s.channels / 2) return fail(FFB_ERR_ARG, "%s: %d pairs of %d channels", s.what, r->pairs, s.channels);
  if (r->pairs == 0 || s.batch == 0 || s.tokens == 0) return FFB_OK;
  if (r->axes < 1 || r->axes > kMaxPositionAxes)
    return fail(FFB_ERR_UNSUPPORTED, "%s: %d axes of positions (1 to %d)", s.what, r->axes, kMaxPositionAxes);
  if (r->position_type < FFB_POSITION_I32 || r->position_type > FFB_POSITION_F32)
    return fail(FFB_ERR_UNSUPPORTED, "%s: position type %d", s.what, r->position_type);
  if (!r->positions || !r->quarters || !r->pair_axes) return fail(FFB_ERR_ARG, "%s: null pointer of the rotary", s.what);
  const uintptr_t width = r->position_type == FFB_POSITION_I64 ? 8 : 4;
  if ((reinterpret_cast<uintptr_t>(r->positions) & (width - 1)) != 0 || (reinterpret_cast<uintptr_t>(r->quarters) & 7u) != 0 ||
      (reinterpret_cast<uintptr_t>(r->pair_axes) & 3u) != 0)
    return fail(FFB_ERR_ARG, "%s: misaligned pointer of the rotary", s.what);
  if (!stride_ok(s.batch, r->batch_stride) || !stride_ok(s.tokens, r->token_stride) || !stride_ok(r->axes, r->axis_stride))
    return fail(FFB_ERR_ARG, "%s: strides of the positions", s.what);
  return FFB_OK;
}

HeadView view(const ffb_heads* h) {
  return h == nullptr ? HeadView{nullptr, 0, 0, 0} : HeadView{h->data, h->batch_stride, h->token_stride, h->head_stride};
}

// Checks one call's tensors (k's NULL together) and fills the kernels' parameters. in: q, k (x); more: dy.
int check_call(const Sizes& s, const ffb_heads* const (&x)[2], const ffb_heads* const (&dy)[2], const ffb_heads* const (&out)[2],
               const ffb_rotary* r, bool backward, HeadsParams* p) {
  static const char *const x_names[2] = {"q", "k"}, *const dy_names[2] = {"q's gradient", "k's gradient"};
  static const char *const out_names[2] = {"q's output", "k's output"};
  int st = check_rotary(s, r);
  if (st != FFB_OK) return st;
  if (x[0] == nullptr) return fail(FFB_ERR_ARG, "%s: q is missing", s.what);
  const int n = x[1] != nullptr ? 2 : 1;
  if (n == 1 && (dy[1] != nullptr || out[1] != nullptr)) return fail(FFB_ERR_ARG, "%s: k is missing", s.what);
  for (int i = 0; i < n; ++i) {
    st = check_view(s, x_names[i], x[i], x[i]->heads);
    if (st == FFB_OK) st = check_view(s, out_names[i], out[i], x[i]->heads);
    if (st == FFB_OK && backward) st = check_view(s, dy_names[i], dy[i], x[i]->heads);
    if (st == FFB_OK) st = check_output(s, out_names[i], *out[i]);
    if (st != FFB_OK) return st;
  }
  for (int i = 0; i < n; ++i) {
    if (empty(s, *out[i])) continue;
    for (int j = 0; j < n; ++j) {
      if (empty(s, *x[j])) continue;
      if (!(i == j && same_view(s, *out[i], *x[j])) && !apart(s, *out[i], *x[j]))
        return fail(FFB_ERR_ARG, "%s: %s overlaps %s", s.what, out_names[i], x_names[j]);
      if (backward && !(i == j && same_view(s, *out[i], *dy[j])) && !apart(s, *out[i], *dy[j]))
        return fail(FFB_ERR_ARG, "%s: %s overlaps %s", s.what, out_names[i], dy_names[j]);
      if (i < j && !apart(s, *out[i], *out[j])) return fail(FFB_ERR_ARG, "%s: the outputs overlap", s.what);
    }
  }
  for (int i = 0; i < 2; ++i) {
    p->x[i] = view(x[i]);
    p->dy[i] = view(dy[i]);
    p->out[i] = view(out[i]);
    p->weight[i] = nullptr;
    p->dweight[i] = nullptr;
    p->heads[i] = i < n ? static_cast<int>(x[i]->heads) : 0;
  }
  p->batch = static_cast<int>(s.batch);
  p->tokens = static_cast<int>(s.tokens);
  p->channels = s.channels;
  p->eps = 0.f;
  p->norm = 0;
  p->rotary = {r->positions, r->position_type, r->axes, r->batch_stride, r->token_stride, r->axis_stride,
               r->quarters, r->pair_axes, r->pairs, r->interleaved != 0, r->inverse != 0};
  return FFB_OK;
}

int check_weights(const char* what, const float* q, const float* k, float eps) {
  if (((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k)) & 15u) != 0) return fail(FFB_ERR_ARG, "%s: misaligned weight", what);
  if (!(eps >= 0.f) || isinf(eps)) return fail(FFB_ERR_ARG, "%s: eps %g", what, static_cast<double>(eps));
  return FFB_OK;
}

bool nothing(const HeadsParams& p) {
  return p.batch == 0 || p.tokens == 0 || (p.heads[0] == 0 && p.heads[1] == 0);
}

}  // namespace

extern "C" {

int ffb_rotary_fwd(const ffb_heads* q, const ffb_heads* k, const ffb_heads* q_out, const ffb_heads* k_out,
                   const ffb_rotary* rotary, int64_t batch, int64_t tokens, int channels, int dtype, void* stream) {
  Sizes s;
  HeadsParams p;
  int st = check_sizes(&s, "rotary", batch, tokens, channels, dtype);
  if (st == FFB_OK) st = check_call(s, {q, k}, {nullptr, nullptr}, {q_out, k_out}, rotary, false, &p);
  if (st != FFB_OK || nothing(p)) return st;
  DeviceInfo info;
  st = device_info(&info);
  if (st != FFB_OK) return st;
  return cuda_status(launch_heads(p, dtype == FFB_F32, as_stream(stream)), "rotary launch");
}

int ffb_qk_norm_rotary_fwd(const ffb_heads* q, const ffb_heads* k, const ffb_heads* q_out, const ffb_heads* k_out,
                           const float* q_weight, const float* k_weight, float eps, const ffb_rotary* rotary,
                           int64_t batch, int64_t tokens, int channels, int dtype, void* stream) {
  Sizes s;
  HeadsParams p;
  int st = check_sizes(&s, "qk_norm_rotary", batch, tokens, channels, dtype);
  if (st == FFB_OK) st = check_weights(s.what, q_weight, k_weight, eps);
  if (st == FFB_OK) st = check_call(s, {q, k}, {nullptr, nullptr}, {q_out, k_out}, rotary, false, &p);
  if (st != FFB_OK || nothing(p)) return st;
  p.weight[0] = q_weight;
  p.weight[1] = k_weight;
  p.eps = eps;
  p.norm = 1;
  DeviceInfo info;
  st = device_info(&info);
  if (st != FFB_OK) return st;
  return cuda_status(launch_heads(p, dtype == FFB_F32, as_stream(stream)), "qk_norm_rotary launch");
}

size_t ffb_qk_norm_rotary_bwd_workspace_bytes(int64_t batch, int64_t tokens, int64_t q_heads, int64_t k_heads,
                                              int channels, int dtype) {
  const int64_t most = (int64_t(1) << 31) - 2;
  if (batch <= 0 || tokens <= 0 || q_heads < 0 || k_heads < 0 || channels <= 0 || channels > kMaxHeadChannels ||
      q_heads > (1 << 20) || k_heads > (1 << 20) || batch > most || tokens > most / batch)
    return 0;
  return heads_bwd_workspace_bytes(batch * tokens, static_cast<int>(q_heads), static_cast<int>(k_heads), channels,
                                   dtype == FFB_F32);
}

int ffb_qk_norm_rotary_bwd(const ffb_heads* dq_out, const ffb_heads* dk_out, const ffb_heads* q, const ffb_heads* k,
                           const ffb_heads* dq, const ffb_heads* dk, const float* q_weight, const float* k_weight,
                           float* dq_weight, float* dk_weight, float eps, const ffb_rotary* rotary, void* workspace,
                           size_t workspace_bytes, int64_t batch, int64_t tokens, int channels, int dtype, void* stream) {
  Sizes s;
  HeadsParams p;
  int st = check_sizes(&s, "qk_norm_rotary_bwd", batch, tokens, channels, dtype);
  if (st == FFB_OK) st = check_weights(s.what, q_weight, k_weight, eps);
  if (st == FFB_OK) st = check_call(s, {q, k}, {dq_out, dk_out}, {dq, dk}, rotary, true, &p);
  if (st != FFB_OK) return st;
  if (((reinterpret_cast<uintptr_t>(dq_weight) | reinterpret_cast<uintptr_t>(dk_weight)) & 3u) != 0)
    return fail(FFB_ERR_ARG, "%s: misaligned weight gradient", s.what);
  if (k == nullptr && dk_weight != nullptr) return fail(FFB_ERR_ARG, "%s: k is missing", s.what);
  DeviceInfo info;
  if (nothing(p)) {
    if (dq_weight == nullptr && dk_weight == nullptr) return FFB_OK;
    st = device_info(&info);
    if (st != FFB_OK) return st;
    cudaError_t e = cudaSuccess;
    if (dq_weight) e = cudaMemsetAsync(dq_weight, 0, sizeof(float) * channels, as_stream(stream));
    if (dk_weight && e == cudaSuccess) e = cudaMemsetAsync(dk_weight, 0, sizeof(float) * channels, as_stream(stream));
    return cuda_status(static_cast<int>(e), "qk_norm_rotary_bwd: zero gradients");
  }
  p.weight[0] = q_weight;
  p.weight[1] = k_weight;
  p.dweight[0] = dq_weight;
  p.dweight[1] = dk_weight;
  p.eps = eps;
  p.norm = 1;
  if (dq_weight != nullptr || dk_weight != nullptr) {
    const size_t need = heads_bwd_workspace_bytes(batch * tokens, p.heads[0], p.heads[1], channels, dtype == FFB_F32);
    if (need > 0 && (!workspace || workspace_bytes < need))
      return fail(FFB_ERR_ARG, "%s: workspace %zu < %zu bytes", s.what, workspace ? workspace_bytes : 0, need);
    if ((reinterpret_cast<uintptr_t>(workspace) & 15u) != 0) return fail(FFB_ERR_ARG, "%s: misaligned workspace", s.what);
  }
  st = device_info(&info);
  if (st != FFB_OK) return st;
  return cuda_status(launch_heads_bwd(p, workspace, dtype == FFB_F32, as_stream(stream)), "qk_norm_rotary_bwd launch");
}

}  // extern "C"
