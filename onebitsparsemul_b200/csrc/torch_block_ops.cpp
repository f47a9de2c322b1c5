// The decoder-block operators of the torch extension `onebit_sparse_cuda`: checks of the tensors, allocation of the outputs and
// the call into the C ABI of libonebitmul. The documented functions are those of onebitsparsemul_b200/block_ops.py, which
// hand their arguments through: in a decode step these calls are a few microseconds of GPU work each, and checks and ctypes
// conversions in Python took longer than that (a norm of one token: 21 us a call from Python through ctypes).
#include <ATen/cuda/CUDAContext.h>
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <cmath>

#include "onebit_sparse_tensor.h"
#include "overlap.h"

namespace {

using torch::Tensor;
using OptTensor = c10::optional<Tensor>;
namespace py = pybind11;

constexpr int64_t kPageTokens = 64;

const Tensor* ptr(const OptTensor& t) { return t.has_value() && t->defined() ? &*t : nullptr; }
void* data(const Tensor* t) { return t ? t->data_ptr() : nullptr; }

[[noreturn]] void raise_library_error(const std::string& message) {
  py::object cls = py::module_::import("onebitsparsemul_b200._lib").attr("OneBitError");
  PyErr_SetString(cls.ptr(), message.c_str());
  throw py::error_already_set();
}
void check_rc(int rc) {
  if (rc != ONEBIT_OK) raise_library_error("libonebitmul error " + std::to_string(rc) + ": " + onebit_last_error());
}

// every tensor on `device`, none of them waiting for a gradient or with a forward-mode tangent
void check_tensors(c10::Device device, std::initializer_list<const Tensor*> tensors) {
  const bool grad = at::GradMode::is_enabled(), tangents = c10::AutogradState::get_tls_state().get_fw_grad_mode();
  for (const Tensor* t : tensors) {
    TORCH_CHECK_VALUE(!t || !grad || !t->requires_grad(), "a tensor wants a gradient, and this operator has none: call it under torch.no_grad()");
    TORCH_CHECK_VALUE(!t || !tangents || !t->_fw_grad(0).defined(), "a tensor has a forward-mode tangent, and this operator has no derivative: give it the primal");
  }
  if (!device.is_cuda()) raise_library_error("no CUDA tensor: this library has no CPU path");
  for (const Tensor* t : tensors) TORCH_CHECK_VALUE(!t || t->device() == device, "tensors on different devices: ", t->device(), " and ", device);
}

int type_code(const Tensor& t) {
  if (t.scalar_type() == torch::kHalf) return ONEBIT_DENSE_F16;
  TORCH_CHECK_TYPE(t.scalar_type() == torch::kBFloat16, "expected float16 or bfloat16, got ", t.scalar_type());
  return ONEBIT_DENSE_BF16;
}

ob_overlap::Place place_of(const Tensor& t) {
  ob_overlap::Place p;
  p.at = reinterpret_cast<uintptr_t>(t.data_ptr()), p.item = (int64_t)t.element_size();
  if (t.is_contiguous()) {
    p.add(p.item, t.numel());
  } else if (t.dim() <= ob_overlap::kMaxDims) {
    for (int64_t d = 0; d < t.dim(); ++d) p.add(t.stride(d) * (int64_t)t.element_size(), t.size(d));
  } else {                                                      // the whole stretch
    for (int64_t d = 0; d < t.dim(); ++d) p.item += t.stride(d) * (int64_t)t.element_size() * (t.size(d) - 1);
  }
  p.empty = t.numel() == 0;
  return p;
}
// every value of one is the same value of the other
bool is_same(const Tensor& a, const Tensor& b) {
  if (a.data_ptr() != b.data_ptr() || a.scalar_type() != b.scalar_type() || a.sizes() != b.sizes()) return false;
  for (int64_t d = 0; d < a.dim(); ++d)
    if (a.size(d) > 1 && a.stride(d) != b.stride(d)) return false;
  return true;
}
// An output has a place of its own for every value, and is an input as a whole or not at all; no part of it is an input that
// other values are computed from (`apart`).
void check_output(const Tensor& out, const char* name, std::initializer_list<const Tensor*> inputs, std::initializer_list<const Tensor*> apart = {}) {
  const ob_overlap::Place place = place_of(out);
  TORCH_CHECK_VALUE(!ob_overlap::may_overlap_itself(place), name, " has several values in one place");
  for (const Tensor* t : inputs)
    TORCH_CHECK_VALUE(!t || is_same(out, *t) || !ob_overlap::may_overlap(place, place_of(*t)), name, " overlaps an input without being it");
  for (const Tensor* t : apart) TORCH_CHECK_VALUE(!t || !ob_overlap::may_overlap(place, place_of(*t)), name, " overlaps an input");
}

// a scalar as the kernels get it
bool finite32(double v) { return std::isfinite((float)v); }

void* stream_of(const Tensor& t) { return at::cuda::getCurrentCUDAStream(t.get_device()).stream(); }

// t as (rows, hidden) with contiguous rows
Tensor rows_of(const Tensor& t, int64_t hidden) {
  Tensor r = t.dim() == 2 ? t : t.reshape({-1, hidden});
  return r.stride(1) == 1 || hidden == 1 ? r : r.contiguous();
}

py::object residual_norm(const Tensor& x, const Tensor& weight, const OptTensor& residual_, const OptTensor& gate_, double residual_scale,
                         const OptTensor& post_, double eps, const OptTensor& out_, const OptTensor& residual_out_) {
  const Tensor *residual = ptr(residual_), *gate = ptr(gate_), *post = ptr(post_), *out = ptr(out_), *residual_out = ptr(residual_out_);
  const int code = type_code(x);
  check_tensors(x.device(), {&x, &weight, residual, gate, post, out, residual_out});
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1 && x.size(-1) <= ONEBIT_NORM_MAX_HIDDEN, "x must be (..., hidden) with 1 <= hidden <= ", ONEBIT_NORM_MAX_HIDDEN);
  const int64_t hidden = x.size(-1);
  const auto channel = [&](const Tensor& t) { return t.dim() == 1 && t.size(0) == hidden; };
  const auto like_x = [&](const Tensor& t) { return t.sizes() == x.sizes(); };
  TORCH_CHECK_VALUE(weight.scalar_type() == x.scalar_type() && channel(weight), "weight must be (", hidden, ",) of x's type");
  TORCH_CHECK_VALUE(!post || (post->scalar_type() == x.scalar_type() && channel(*post)), "post_weight must be (", hidden, ",) of x's type");
  TORCH_CHECK_VALUE(finite32(eps) && eps >= 0 && finite32(residual_scale), "eps must be finite and not negative, residual_scale finite (in 32 bits)");
  Tensor h, r2;
  if (!residual) {
    TORCH_CHECK_VALUE(!gate && !post && !residual_out && residual_scale == 1.0, "gate, post_weight, residual_scale and residual_out need a residual");
  } else {
    TORCH_CHECK_VALUE(like_x(*residual) && (residual->scalar_type() == x.scalar_type() || residual->scalar_type() == torch::kFloat),
                      "residual must have x's shape and x's type or float32");
    TORCH_CHECK_VALUE(!residual_out || (like_x(*residual_out) && residual_out->scalar_type() == residual->scalar_type() && residual_out->is_contiguous()),
                      "residual_out must be contiguous with residual's shape and type");
    h = residual_out ? *residual_out : torch::empty(x.sizes(), residual->options());
    r2 = rows_of(*residual, hidden);
  }
  // the weights are read for every row, and weight after h is written
  if (out) check_output(*out, "out", {&x, residual, gate, residual_out}, {&weight, post});
  if (residual_out) check_output(*residual_out, "residual_out", {&x, residual, gate}, {&weight, post});
  TORCH_CHECK_VALUE(!out || !residual_out || out->numel() == 0 || out->data_ptr() != residual_out->data_ptr(), "out and residual_out must be different tensors");
  Tensor g2;
  int64_t gate_stride = 0;
  if (gate) {
    TORCH_CHECK_VALUE(gate->scalar_type() == x.scalar_type() && (channel(*gate) || like_x(*gate)), "gate must be (hidden,) or x's shape, of x's type");
    const bool per_row = like_x(*gate) && gate->dim() > 1;
    g2 = per_row ? rows_of(*gate, hidden) : gate->contiguous();
    gate_stride = per_row ? g2.stride(0) : 0;
  }
  TORCH_CHECK_VALUE(!out || (like_x(*out) && out->scalar_type() == x.scalar_type() && out->is_contiguous()), "out must be contiguous with x's shape and type");
  Tensor y = out ? *out : torch::empty(x.sizes(), x.options());
  const Tensor x2 = rows_of(x, hidden), w = weight.contiguous(), p = post ? post->contiguous() : Tensor();
  if (x2.size(0) > 0) {
    c10::cuda::CUDAGuard guard(x.device());
    check_rc(onebit_residual_norm(x2.data_ptr(), x2.stride(0), residual ? r2.data_ptr() : nullptr, residual ? r2.stride(0) : 0,
                                  residual && r2.scalar_type() == torch::kFloat, gate ? g2.data_ptr() : nullptr, gate_stride, post ? p.data_ptr() : nullptr,
                                  w.data_ptr(), y.data_ptr(), hidden, residual ? h.data_ptr() : nullptr, hidden, x2.size(0), hidden, (float)residual_scale,
                                  (float)eps, code, stream_of(x)));
  }
  return residual ? py::object(py::make_tuple(y, h)) : py::cast(y);
}

void check_heads(const Tensor& t, const char* name, int64_t tokens, int64_t heads, int64_t dim) {   // -1: any
  TORCH_CHECK_VALUE(t.dim() == 3 && (tokens < 0 || t.size(0) == tokens) && (heads < 0 || t.size(1) == heads) && (dim < 0 || t.size(2) == dim), name, " must be (",
                    tokens < 0 ? "?" : std::to_string(tokens), ", ", heads < 0 ? "?" : std::to_string(heads), ", ", dim < 0 ? "?" : std::to_string(dim), "), got ", t.sizes());
}
Tensor inner_contiguous(const Tensor& t) { return t.stride(2) == 1 || t.size(2) == 1 ? t : t.contiguous(); }

bool interleaved_layout(const std::string& layout) {
  TORCH_CHECK_VALUE(layout == "half" || layout == "interleaved", "layout must be 'half' or 'interleaved', got '", layout, "'");
  return layout == "interleaved";
}
int rotary_dim_of(const Tensor& inv_freq, int64_t head_dim) {
  TORCH_CHECK_VALUE(inv_freq.scalar_type() == torch::kDouble && inv_freq.dim() == 1 && inv_freq.is_contiguous(),
                    "inv_freq must be a contiguous float64 vector (32 bits lose the angles of far positions)");
  TORCH_CHECK_VALUE(2 * inv_freq.numel() <= head_dim, inv_freq.numel(), " pairs do not fit a head of ", head_dim);
  return (int)(2 * inv_freq.numel());
}
void check_turned(const Tensor& out, const Tensor& x, const char* name, std::initializer_list<const Tensor*> apart) {
  TORCH_CHECK_VALUE(out.sizes() == x.sizes() && out.scalar_type() == x.scalar_type() && (out.stride(2) == 1 || out.size(2) == 1), name,
                    " must have the input's shape and type and contiguous heads");
  check_output(out, name, {&x}, apart);
}

Tensor rotary_tokens(const Tensor& x, const Tensor& positions, const Tensor& inv_freq, const std::string& layout, double magnitude, const OptTensor& out_) {
  const Tensor* out = ptr(out_);
  const int code = type_code(x);
  check_tensors(x.device(), {&x, &positions, &inv_freq, out});
  check_heads(x, "x", -1, -1, -1);
  const int64_t tokens = x.size(0), heads = x.size(1), dim = x.size(2);
  TORCH_CHECK_VALUE(dim >= 1 && dim <= ONEBIT_ROTARY_MAX_DIM && heads >= 1 && heads <= 4096 && tokens <= (1 << 24), "x must be (tokens <= 2^24, heads <= 4096, head_dim <= ",
                    ONEBIT_ROTARY_MAX_DIM, ")");
  const bool wide = positions.scalar_type() == torch::kLong;
  TORCH_CHECK_VALUE((wide || positions.scalar_type() == torch::kInt) && positions.dim() == 1 && positions.size(0) == tokens, "positions must be (tokens,) int32 or int64");
  const bool inter = interleaved_layout(layout);
  TORCH_CHECK_VALUE(finite32(magnitude), "magnitude must be finite (in 32 bits)");
  const int rotary_dim = rotary_dim_of(inv_freq, dim);
  if (out) check_turned(*out, x, "out", {&positions, &inv_freq});
  Tensor y = out ? *out : torch::empty(x.sizes(), x.options());
  if (tokens > 0) {
    const Tensor x1 = inner_contiguous(x), p = positions.contiguous();
    c10::cuda::CUDAGuard guard(x.device());
    check_rc(onebit_rotary(x1.data_ptr(), x1.stride(0), x1.stride(1), y.data_ptr(), y.stride(0), y.stride(1), p.data_ptr(), wide, inv_freq.data_ptr<double>(),
                           rotary_dim, inter, (float)magnitude, tokens, heads, dim, code, stream_of(x)));
  }
  return y;
}

// (pages, kv_heads, head_dim) of a cache's tensors
std::tuple<int64_t, int64_t, int64_t> check_cache(const Tensor& k_pages, const Tensor& v_pages, const Tensor& k_scale, const Tensor& v_scale) {
  TORCH_CHECK_VALUE(k_pages.dim() == 4 && k_pages.size(2) == kPageTokens && (k_pages.size(3) == 64 || k_pages.size(3) == 128), "k_pages must be (pages, kv_heads, 64, 64 or 128)");
  const int64_t pages = k_pages.size(0), heads = k_pages.size(1), dim = k_pages.size(3);
  const auto scale_shape = [&](const Tensor& t) { return t.dim() == 2 && t.size(0) == pages && t.size(1) == heads; };
  TORCH_CHECK_VALUE(v_pages.dim() == 4 && v_pages.size(0) == pages && v_pages.size(1) == heads && v_pages.size(2) == dim && v_pages.size(3) == kPageTokens &&
                        scale_shape(k_scale) && scale_shape(v_scale),
                    "with ", pages, " pages of ", heads, " heads of ", dim, ": v_pages must be (", pages, ", ", heads, ", ", dim, ", 64), scales (", pages, ", ", heads, ")");
  TORCH_CHECK_TYPE(k_pages.scalar_type() == torch::kFloat8_e4m3fn && v_pages.scalar_type() == torch::kFloat8_e4m3fn && k_scale.scalar_type() == torch::kFloat &&
                       v_scale.scalar_type() == torch::kFloat,
                   "pages must be float8_e4m3fn, scales float32");
  for (const Tensor* t : {&k_pages, &v_pages, &k_scale, &v_scale})
    TORCH_CHECK_VALUE(t->is_contiguous() && t->device() == k_pages.device(), "pages and scales must be contiguous, on one device");
  TORCH_CHECK_VALUE(pages >= 1 && heads >= 1 && heads <= 4096, "need at least one page and 1 to 4096 heads");
  const ob_overlap::Place places[] = {place_of(k_pages), place_of(v_pages), place_of(k_scale), place_of(v_scale)};
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < i; ++j) TORCH_CHECK_VALUE(!ob_overlap::may_overlap(places[i], places[j]), "pages and scales must be four tensors that share no memory");
  return {pages, heads, dim};
}

// (sequences, width) of a batch's tensors
std::tuple<int64_t, int64_t> check_batch(const Tensor& q_start, const Tensor& kv_len, const Tensor& table) {
  TORCH_CHECK_TYPE(q_start.scalar_type() == torch::kInt && kv_len.scalar_type() == torch::kInt && table.scalar_type() == torch::kInt, "q_start, kv_len and block_table must be int32");
  TORCH_CHECK_VALUE(table.dim() == 2 && table.size(0) >= 1 && table.size(1) >= 1 && (table.stride(1) == 1 || table.size(1) == 1),
                    "block_table must be (sequences, width), at least 1 x 1, with contiguous rows");
  const int64_t seqs = table.size(0), width = table.size(1);
  TORCH_CHECK_VALUE(q_start.dim() == 1 && q_start.size(0) == seqs + 1 && kv_len.dim() == 1 && kv_len.size(0) == seqs && q_start.is_contiguous() && kv_len.is_contiguous(),
                    "with ", seqs, " sequences: q_start must be (", seqs + 1, ",), kv_len (", seqs, ",), both contiguous");
  TORCH_CHECK_VALUE(q_start.device() == table.device() && kv_len.device() == table.device(), "q_start, kv_len and block_table must be on one device");
  TORCH_CHECK_VALUE(seqs <= (1 << 16) && width <= (1 << 24), "at most 2^16 sequences of 2^24 pages");
  return {seqs, width};
}

py::object cache_append(const Tensor& k, const Tensor& v, const Tensor& k_pages, const Tensor& v_pages, const Tensor& k_scale, const Tensor& v_scale,
                        const Tensor& q_start, const Tensor& kv_len, const Tensor& table, int64_t max_new, const OptTensor& q_, const OptTensor& inv_freq_,
                        const std::string& layout, double magnitude, const OptTensor& q_out_) {
  const Tensor *q = ptr(q_), *inv_freq = ptr(inv_freq_), *q_out = ptr(q_out_);
  const int code = type_code(k);
  check_tensors(k.device(), {&k, &v, q, inv_freq, q_out, &k_pages, &k_scale, &v_scale, &table});
  const int64_t H = k_pages.size(1), D = k_pages.size(3), tokens = k.dim() == 3 ? k.size(0) : -1;
  check_heads(k, "k", -1, H, D);
  check_heads(v, "v", tokens, H, D);
  TORCH_CHECK_TYPE(v.scalar_type() == k.scalar_type() && (!q || q->scalar_type() == k.scalar_type()), "q, k and v must have one type");
  TORCH_CHECK_VALUE(tokens <= (1 << 24), "at most 2^24 tokens");
  const bool inter = interleaved_layout(layout);
  TORCH_CHECK_VALUE(finite32(magnitude), "magnitude must be finite (in 32 bits)");
  const int rotary_dim = inv_freq ? rotary_dim_of(*inv_freq, D) : 0;
  int64_t heads = H;
  Tensor y, q1;
  if (q) {
    check_heads(*q, "q", tokens, -1, D);
    heads = q->size(1);
    TORCH_CHECK_VALUE(inv_freq, "q is only turned: it needs inv_freq");
    TORCH_CHECK_VALUE(heads % H == 0 && heads >= 1 && heads <= 4096, heads, " query heads are no multiple of ", H, " cache heads");
    if (q_out) check_turned(*q_out, *q, "q_out", {&k, &v, inv_freq, &k_pages, &v_pages, &k_scale, &v_scale, &q_start, &kv_len, &table});
    y = q_out ? *q_out : torch::empty(q->sizes(), q->options());
    q1 = inner_contiguous(*q);
  } else {
    TORCH_CHECK_VALUE(!q_out, "q_out without q");
  }
  if (tokens > 0) {
    const Tensor k1 = inner_contiguous(k), v1 = inner_contiguous(v);
    c10::cuda::CUDAGuard guard(k.device());
    check_rc(onebit_cache_append_ex(k1.data_ptr(), k1.stride(0), k1.stride(1), v1.data_ptr(), v1.stride(0), v1.stride(1), q ? q1.data_ptr() : nullptr, q ? q1.stride(0) : 0,
                                 q ? q1.stride(1) : 0, q ? y.data_ptr() : nullptr, q ? y.stride(0) : 0, q ? y.stride(1) : 0,
                                 static_cast<const double*>(data(inv_freq)), rotary_dim, inter, (float)magnitude, k_pages.data_ptr(), v_pages.data_ptr(),
                                 k_scale.data_ptr<float>(), v_scale.data_ptr<float>(), k_pages.size(0), q_start.data_ptr<int>(), kv_len.data_ptr<int>(),
                                 table.data_ptr<int>(), table.stride(0), table.size(1), tokens, table.size(0), heads, H, D, max_new, code, stream_of(k)));
  }
  return q ? py::cast(y) : py::none();
}

Tensor cache_attend(const Tensor& q, const Tensor& k_pages, const Tensor& v_pages, const Tensor& k_scale, const Tensor& v_scale, const Tensor& q_start,
                    const Tensor& kv_len, const Tensor& table, int64_t max_new, const c10::optional<double>& scale_, bool causal, const OptTensor& out_) {
  const Tensor* out = ptr(out_);
  const int code = type_code(q);
  check_tensors(q.device(), {&q, out, &k_pages, &k_scale, &v_scale, &table});
  const int64_t H = k_pages.size(1), D = k_pages.size(3);
  check_heads(q, "q", -1, -1, D);
  const int64_t tokens = q.size(0), heads = q.size(1);
  TORCH_CHECK_VALUE(heads % H == 0 && heads >= 1 && heads <= 4096, heads, " query heads are no multiple of ", H, " cache heads");
  TORCH_CHECK_VALUE(tokens <= (1 << 24), "at most 2^24 tokens");
  const double scale = scale_.has_value() ? *scale_ : 1.0 / std::sqrt((double)D);
  TORCH_CHECK_VALUE(finite32(scale), "scale must be finite (in 32 bits)");
  const auto aligned = [](const Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; };
  TORCH_CHECK_VALUE(!out || (out->sizes() == q.sizes() && out->scalar_type() == q.scalar_type() && out->is_contiguous() && aligned(*out)),
                    "out must be contiguous (and 16-byte aligned) with q's shape and type");
  if (out) check_output(*out, "out", {}, {&q, &k_pages, &v_pages, &k_scale, &v_scale, &q_start, &kv_len, &table});
  Tensor y = out ? *out : torch::empty(q.sizes(), q.options());
  if (tokens > 0) {
    const bool as_it_is = q.stride(2) == 1 && q.stride(0) % 8 == 0 && q.stride(1) % 8 == 0 && aligned(q);
    const Tensor q1 = as_it_is ? q : q.clone(at::MemoryFormat::Contiguous);
    c10::cuda::CUDAGuard guard(q.device());
    const int64_t need = (int64_t)onebit_cache_attend_workspace(table.size(1), tokens, table.size(0), heads, H, D, max_new);
    const Tensor ws = need > 0 ? torch::empty({need}, q.options().dtype(torch::kUInt8)) : Tensor();
    check_rc(onebit_cache_attend(q1.data_ptr(), q1.stride(0), q1.stride(1), y.data_ptr(), heads * D, D, k_pages.data_ptr(), v_pages.data_ptr(), k_scale.data_ptr<float>(),
                                 v_scale.data_ptr<float>(), k_pages.size(0), q_start.data_ptr<int>(), kv_len.data_ptr<int>(), table.data_ptr<int>(), table.stride(0),
                                 table.size(1), tokens, table.size(0), heads, H, D, max_new, (float)scale, causal, code, need > 0 ? ws.data_ptr() : nullptr, (size_t)need,
                                 stream_of(q)));
  }
  return y;
}

}  // namespace

void bind_block_ops(py::module_& m) {
  m.def("residual_norm", &residual_norm);
  m.def("rotary_tokens", &rotary_tokens);
  m.def("check_cache", &check_cache);
  m.def("check_batch", &check_batch);
  m.def("cache_append", &cache_append);
  m.def("cache_attend", &cache_attend);
}
