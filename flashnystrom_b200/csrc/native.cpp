// The eager path of flash_nystrom_attention and of the module in C++: argument checks, allocations, the autograd nodes and the
// calls of the C ABI.  Host time of a forward and backward pass (us, the autograd functions in Python / this): the op 185 / 111,
// with the convolution residual 340 / 150 (about 50 of each are the launches), the module at B=4, N=4096, 8 heads of 64
// 816 / 466; inference through the op 48 / 24.  (A pass of that module among others: 793 / 479.)
//
// attention() only takes calls that it can see through completely: plain CUDA tensors of one device and dtype in one of the
// two layouts, no dispatch mode, no forward-mode tangent (tracing and functorch transforms the caller sees).  For anything
// else it returns nothing and the caller goes on in Python, which accepts or refuses it as ever.
#include <torch/extension.h>

#include <ATen/TensorSubclassLikeUtils.h>
#include <ATen/autocast_mode.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

#include <atomic>
#include <cmath>
#include <cstdlib>

#include "../../include/flashnystrom_b200.h"

namespace {

using torch::autograd::AutogradContext;
using torch::autograd::Variable;
using torch::autograd::variable_list;

std::atomic<uint32_t> g_flags{0};
PyObject* g_debug = nullptr;     // called with (dO, dQ, dK, dV, step2, k2inv) when FNB_BWD_DEBUG is set

void check(int rc) { TORCH_CHECK(rc == 0, "flashnystrom_b200: ", fnb_last_error(), " (status ", rc, ")"); }

constexpr int kNoLayout = -1;
int layout_of(const at::Tensor& t) {
  if (t.is_contiguous()) return FNB_LAYOUT_BHND;
  return t.transpose(1, 2).is_contiguous() ? FNB_LAYOUT_BNHD : kNoLayout;
}
int dtype_of(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return FNB_F32;
    case at::kHalf: return FNB_F16;
    case at::kBFloat16: return FNB_BF16;
    default: return -1;
  }
}
// shapes that take the (B, N, H, D) layout: the tensor-core kernels' own
bool takes_bnhd(int dtype, int64_t D, int64_t m, uint32_t flags) {
  return !(flags & FNB_FLAG_FORCE_GENERIC) && dtype != FNB_F32 && ((D == 64 && m <= 64) || (D == 128 && m <= 128));
}
at::Tensor empty_in(const at::Tensor& like, int layout) {
  const int64_t B = like.size(0), H = like.size(1), N = like.size(2), D = like.size(3);
  return layout == FNB_LAYOUT_BNHD ? at::empty_strided({B, H, N, D}, {N * H * D, D, H * D, 1}, like.options())
                                   : at::empty({B, H, N, D}, like.options());
}
at::Tensor to_layout(const at::Tensor& t, int layout) {
  if (layout_of(t) == layout) return t;
  return layout == FNB_LAYOUT_BNHD ? t.transpose(1, 2).contiguous().transpose(1, 2) : t.contiguous();
}

// The FP32 tensors that the backward needs, in one buffer: lse1, q~, k~, K2, lse2, iterates, K2inv, Bmat, lse3, step2 (the order of
// fnb_fwd_args), each on a 256-byte step.
struct Saved {
  int64_t offset[10], floats;
  Saved(int64_t BH, int64_t N, int64_t D, int64_t m, int64_t J) {
    const int64_t n[10] = {N, m * D, m * D, m * m, m, (J + 1) * m * m, m * m, m * D, m, m * D};
    floats = 0;
    for (int i = 0; i < 10; ++i) {
      offset[i] = floats;
      floats += (BH * n[i] + 63) / 64 * 64;
    }
  }
};

struct Call {
  fnb_shape shape;
  int layout;
  at::Tensor status;       // the device's status word
};
fnb_shape shape_of(at::IntArrayRef sizes, int dtype, int64_t m, int64_t J, double kappa, int layout, uint32_t flags) {
  fnb_shape s{};
  s.batch = sizes[0]; s.heads = sizes[1]; s.seq_len = sizes[2]; s.head_dim = (int32_t)sizes[3];
  s.num_landmarks = (int32_t)m; s.newton_iter = (int32_t)J; s.dtype = dtype;
  s.kappa_star = (float)kappa; s.flags = flags; s.layout = layout;
  return s;
}
at::Tensor bytes(size_t n, const at::Tensor& like) {
  return at::empty({(int64_t)std::max<size_t>(n, 256)}, like.options().dtype(at::kByte));
}
// (with the tensors' device current: workspace sizes follow its SM count)
at::Tensor run_forward(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const Call& c, at::Tensor& saved) {
  const Saved parts(c.shape.batch * c.shape.heads, c.shape.seq_len, c.shape.head_dim, c.shape.num_landmarks, c.shape.newton_iter);
  at::Tensor out = empty_in(q, c.layout);
  saved = at::empty({parts.floats}, q.options().dtype(at::kFloat));
  at::Tensor ws = bytes(fnb_fwd_workspace_bytes(&c.shape), q);
  float* s = saved.data_ptr<float>();
  fnb_fwd_args a{};
  a.shape = c.shape;
  a.q = q.data_ptr(); a.k = k.data_ptr(); a.v = v.data_ptr(); a.out = out.data_ptr();
  float** to[10] = {&a.lse1, &a.q_landmarks, &a.k_landmarks, &a.k2, &a.lse2, &a.ns_iterates, &a.k2_inv, &a.bmat, &a.lse3, &a.step2};
  for (int i = 0; i < 10; ++i) *to[i] = s + parts.offset[i];
  a.workspace = ws.data_ptr(); a.workspace_bytes = (size_t)ws.numel();
  a.device = q.device().index();
  a.stream = c10::cuda::getCurrentCUDAStream(q.device().index()).stream();
  a.device_status = c.status.data_ptr<int32_t>();
  check(fnb_forward(&a));
  return out;
}

at::Tensor run_conv(const at::Tensor& v, int layout, const at::Tensor& w32, const at::Tensor* base, bool transposed) {
  at::Tensor result = empty_in(v, layout);
  fnb_conv_args a{};
  a.batch = v.size(0); a.heads = v.size(1); a.seq_len = v.size(2); a.head_dim = (int32_t)v.size(3);
  a.kernel_size = (int32_t)w32.size(1); a.dtype = dtype_of(v); a.layout = layout;
  a.v = v.data_ptr(); a.base = base ? base->data_ptr() : nullptr; a.result = result.data_ptr(); a.weight = w32.data_ptr<float>();
  a.transposed = transposed ? 1 : 0; a.device = v.device().index();
  a.stream = c10::cuda::getCurrentCUDAStream(v.device().index()).stream();
  check(fnb_conv_residual(&a));
  return result;
}
at::Tensor run_conv_dweight(const at::Tensor& v, const at::Tensor& g, int layout, int64_t ks) {
  at::Tensor dw = at::empty({v.size(1), ks}, v.options().dtype(at::kFloat));
  at::Tensor ws = bytes(fnb_conv_dweight_workspace_bytes(v.size(0), v.size(1), v.size(2), (int32_t)ks), v);
  fnb_conv_dw_args a{};
  a.batch = v.size(0); a.heads = v.size(1); a.seq_len = v.size(2); a.head_dim = (int32_t)v.size(3);
  a.kernel_size = (int32_t)ks; a.dtype = dtype_of(v); a.layout = layout;
  a.v = v.data_ptr(); a.d_out = g.data_ptr(); a.d_weight = dw.data_ptr<float>();
  a.workspace = ws.data_ptr(); a.workspace_bytes = (size_t)ws.numel(); a.device = v.device().index();
  a.stream = c10::cuda::getCurrentCUDAStream(v.device().index()).stream();
  check(fnb_conv_residual_dweight(&a));
  return dw;
}
// the taps take part rounded to the tensors' dtype
at::Tensor rounded_taps(const at::Tensor& weight, const at::Tensor& v) {
  return weight.detach().to(v.scalar_type()).to(at::kFloat).contiguous();
}

// Attention, with the convolution residual where a weight is given (its gradient with respect to v is then added to the
// attention's in the convolution kernel).
struct AttentionNode : torch::autograd::Function<AttentionNode> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                            const std::optional<at::Tensor>& weight, const Call& c) {
    at::Tensor saved;
    at::Tensor out = run_forward(q, k, v, c, saved);
    // (a gradient of the taps alone needs v and nothing else of the attention)
    const bool inputs = q.requires_grad() || k.requires_grad() || v.requires_grad();
    variable_list keep = inputs ? variable_list{v, q, k, saved} : variable_list{v};
    if (weight) {
      at::Tensor w32 = rounded_taps(*weight, v);
      out = run_conv(v, c.layout, w32, &out, false);
      keep.push_back(w32);
      ctx->saved_data["weight_dtype"] = (int64_t)weight->scalar_type();
    }
    ctx->save_for_backward(keep);
    ctx->saved_data["conv"] = weight.has_value();
    ctx->saved_data["m"] = (int64_t)c.shape.num_landmarks;
    ctx->saved_data["J"] = (int64_t)c.shape.newton_iter;
    ctx->saved_data["kappa"] = (double)c.shape.kappa_star;
    ctx->saved_data["status"] = c.status;
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list kept = ctx->get_saved_variables();
    const bool conv = ctx->saved_data["conv"].toBool(), inputs = kept.size() > 2;
    const at::Tensor& v = kept[0];
    at::Tensor g = grads[0];
    TORCH_CHECK(g.defined() && g.is_cuda() && g.dim() == 4, "dO must be a 4D CUDA tensor (flashnystrom_b200 has no CPU path)");
    const int dtype = dtype_of(g);
    TORCH_CHECK(dtype >= 0, "Supported dtypes: float32, float16, bfloat16");
    c10::cuda::CUDAGuard guard(g.device());
    const int64_t m = ctx->saved_data["m"].toInt();
    const uint32_t flags = g_flags.load();
    int layout = layout_of(v);
    if (layout != FNB_LAYOUT_BNHD || !takes_bnhd(dtype, g.size(3), m, flags)) layout = FNB_LAYOUT_BHND;
    g = to_layout(g, layout);
    for (size_t i = 0; i < (inputs ? 3 : 1); ++i)
      TORCH_CHECK(kept[i].scalar_type() == g.scalar_type() && kept[i].device() == g.device() && kept[i].sizes() == g.sizes() &&
                      layout_of(kept[i]) == layout,
                  "a saved q, k or v does not match dO in shape, dtype, device or layout");
    variable_list result(5);
    if (inputs) attention_backward(ctx, kept[1], kept[2], v, kept[3], g, layout, m, flags, result);
    if (conv) {
      const at::Tensor& w32 = kept.back();
      TORCH_CHECK(w32.scalar_type() == at::kFloat && w32.device() == g.device() && w32.dim() == 2 && w32.size(0) == g.size(1) && w32.is_contiguous(),
                  "the saved convolution weights do not match dO");
      if (ctx->needs_input_grad(2)) result[2] = run_conv(g, layout, w32, &result[2], true);
      if (ctx->needs_input_grad(3))
        result[3] = run_conv_dweight(v, g, layout, w32.size(1)).to((at::ScalarType)ctx->saved_data["weight_dtype"].toInt());
    }
    return result;
  }

  static void attention_backward(AutogradContext* ctx, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, at::Tensor saved,
                                 const at::Tensor& g, int layout, int64_t m, uint32_t flags, variable_list& result) {
    const int64_t J = ctx->saved_data["J"].toInt();
    const Saved parts(g.size(0) * g.size(1), g.size(2), g.size(3), m, J);
    TORCH_CHECK(saved.device() == g.device() && saved.scalar_type() == at::kFloat && saved.dim() == 1 && saved.numel() == parts.floats &&
                    saved.is_contiguous(),
                "the saved tensors do not match dO");
    if (reinterpret_cast<uintptr_t>(saved.data_ptr()) & 15u) saved = saved.clone();   // (a saved-tensor hook may hand it back anywhere)
    const at::Tensor status = ctx->saved_data["status"].toTensor();
    fnb_bwd_args a{};
    a.shape = shape_of(g.sizes(), dtype_of(g), m, J, ctx->saved_data["kappa"].toDouble(), layout, flags);
    check(fnb_check_shape(&a.shape));
    at::Tensor dq = empty_in(g, layout), dk = empty_in(g, layout), dv = empty_in(g, layout);
    at::Tensor ws = bytes(fnb_bwd_workspace_bytes(&a.shape), g);
    const float* s = saved.data_ptr<float>();
    a.q = q.data_ptr(); a.k = k.data_ptr(); a.v = v.data_ptr(); a.d_out = g.data_ptr();
    a.lse1 = s + parts.offset[0]; a.q_landmarks = s + parts.offset[1]; a.k_landmarks = s + parts.offset[2]; a.k2 = s + parts.offset[3];
    a.ns_iterates = s + parts.offset[5]; a.k2_inv = s + parts.offset[6]; a.bmat = s + parts.offset[7]; a.lse3 = s + parts.offset[8];
    a.step2 = s + parts.offset[9];
    a.dq = dq.data_ptr(); a.dk = dk.data_ptr(); a.dv = dv.data_ptr();
    a.workspace = ws.data_ptr(); a.workspace_bytes = (size_t)ws.numel(); a.device = g.device().index();
    a.stream = c10::cuda::getCurrentCUDAStream(g.device().index()).stream();
    a.device_status = status.data_ptr<int32_t>();
    check(fnb_backward(&a));
    if (std::getenv("FNB_BWD_DEBUG") && std::getenv("FNB_BWD_DEBUG")[0] && g_debug) {
      py::gil_scoped_acquire gil;
      const int64_t BH = g.size(0) * g.size(1), D = g.size(3);
      py::reinterpret_borrow<py::object>(g_debug)(g, dq, dk, dv, saved.narrow(0, parts.offset[9], BH * m * D),
                                                  saved.narrow(0, parts.offset[6], BH * m * m));
    }
    result[0] = dq;
    result[1] = dk;
    result[2] = dv;
  }
};

// The three projections of the module as one node.  q, k and v come out as the (B, H, N, D) views of (B, N, H D) products; the
// backward is written in differentiable operators, as that of three torch linears is, with the gradients of x added up in the
// products.
at::Tensor head_split(const at::Tensor& x2, const at::Tensor& w, int64_t B, int64_t N, int64_t H) {
  const int64_t dim = w.size(0), D = dim / H;
  at::Tensor t = at::empty_strided({B, H, N, D}, {N * dim, D, dim, 1}, x2.options());
  at::Tensor flat = t.as_strided({B * N, dim}, {dim, 1});
  at::mm_out(flat, x2, w.t());
  return t;
}
at::Tensor rows_of(const at::Tensor& t) { return t.transpose(1, 2).reshape({t.size(0) * t.size(2), t.size(1) * t.size(3)}); }

// Both nodes keep what a gradient that is wanted takes, as a torch linear does: its input for the weight's, its weight for the
// input's.  (The rest may be changed in place, and is not held.)
bool wants(const at::Tensor& t) { return t.requires_grad(); }
at::Tensor kept_if(bool keep, const at::Tensor& t) { return keep ? t : at::Tensor(); }

struct ProjectionsNode : torch::autograd::Function<ProjectionsNode> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& wq, const at::Tensor& wk, const at::Tensor& wv,
                               int64_t H) {
    const int64_t B = x.size(0), N = x.size(1);
    const at::Tensor x2 = x.view({B * N, x.size(2)});
    ctx->save_for_backward({kept_if(wants(wq) || wants(wk) || wants(wv), x), kept_if(wants(x), wq), kept_if(wants(x), wk), kept_if(wants(x), wv)});
    return {head_split(x2, wq, B, N, H), head_split(x2, wk, B, N, H), head_split(x2, wv, B, N, H)};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list kept = ctx->get_saved_variables();
    const at::Tensor x2 = kept[0].defined() ? kept[0].reshape({-1, kept[0].size(-1)}) : at::Tensor();
    variable_list result(5);
    at::Tensor dx;
    for (int i = 0; i < 3; ++i) {
      const at::Tensor g = rows_of(grads[i]);
      if (ctx->needs_input_grad(0)) dx = i == 0 ? at::mm(g, kept[1]) : at::addmm(dx, g, kept[1 + i]);
      if (ctx->needs_input_grad(1 + i)) result[1 + i] = at::mm(g.t(), x2);
    }
    if (dx.defined()) result[0] = dx.view({grads[0].size(0), grads[0].size(2), dx.size(1)});
    return result;
  }
};

// The output projection of (B, H, N, D) tensors, likewise.
at::Tensor project_out(const at::Tensor& o, const at::Tensor& w) {
  return at::mm(rows_of(o), w.t()).view({o.size(0), o.size(2), w.size(0)});
}
struct OutputNode : torch::autograd::Function<OutputNode> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& o, const at::Tensor& w) {
    ctx->save_for_backward({kept_if(wants(w), o), kept_if(wants(o), w)});
    ctx->saved_data["heads"] = o.size(1);
    at::Tensor y = at::empty({o.size(0), o.size(2), w.size(0)}, o.options());
    at::Tensor flat = y.as_strided({o.size(0) * o.size(2), w.size(0)}, {w.size(0), 1});
    at::mm_out(flat, rows_of(o), w.t());
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list kept = ctx->get_saved_variables();
    const at::Tensor &o = kept[0], &w = kept[1];
    const int64_t B = grads[0].size(0), N = grads[0].size(1), H = ctx->saved_data["heads"].toInt();
    const at::Tensor g = grads[0].reshape({B * N, -1});
    variable_list result(2);
    if (ctx->needs_input_grad(0)) result[0] = at::mm(g, w).view({B, N, H, w.size(1) / H}).transpose(1, 2);
    if (ctx->needs_input_grad(1)) result[1] = at::mm(g.t(), rows_of(o));
    return result;
  }
};

bool plain(const at::Tensor& t) { return t.is_cuda() && t.layout() == at::kStrided && !at::isTensorSubclassLike(t) && !t.is_neg() && !t.is_conj(); }
bool has_tangent(const at::Tensor& t) { return t._fw_grad(0).defined(); }

// taps for B x H slices
bool takes_taps(const at::Tensor& w, const at::Tensor& like, int64_t B, int64_t H) {
  return plain(w) && w.device() == like.device() && at::isFloatingType(w.scalar_type()) && w.dim() == 2 && w.size(0) == H && w.size(1) % 2 == 1 &&
         w.size(1) <= 127 && !has_tangent(w) && B * H <= 65535;
}
bool takes_numbers(int64_t m, int64_t J, double kappa) {
  return m >= 1 && m <= INT32_MAX && J >= 1 && J <= INT32_MAX && std::isfinite(kappa);
}

// (without the interpreter's lock, with the tensors' device current, all of it checked)
at::Tensor run_attention(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const std::optional<at::Tensor>& weight, const Call& c) {
  if (at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad() || (weight && weight->requires_grad())))
    return AttentionNode::apply(q, k, v, weight, c);
  at::Tensor saved;
  at::Tensor out = run_forward(q, k, v, c, saved);
  return weight ? run_conv(v, c.layout, rounded_taps(*weight, v), &out, false) : out;
}

// out, or nothing where the call is not one for this path
std::optional<at::Tensor> attention(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, int64_t m, int64_t J, double kappa,
                                    const std::optional<at::Tensor>& weight, const at::Tensor& status) {
  if (c10::impl::dispatch_mode_enabled()) return std::nullopt;
  for (const at::Tensor* t : {&q, &k, &v})
    if (!plain(*t) || t->dim() != 4 || t->scalar_type() != q.scalar_type() || t->sizes() != q.sizes() || t->device() != q.device() || has_tangent(*t))
      return std::nullopt;
  const int dtype = dtype_of(q);
  if (dtype < 0 || q.numel() == 0 || !takes_numbers(m, J, kappa)) return std::nullopt;
  if (status.device() != q.device()) return std::nullopt;
  const uint32_t flags = g_flags.load();
  int layout = layout_of(q);
  if (layout == FNB_LAYOUT_BNHD && !takes_bnhd(dtype, q.size(3), m, flags)) return std::nullopt;
  if (layout == kNoLayout || layout_of(k) != layout || layout_of(v) != layout) return std::nullopt;
  if (weight && !takes_taps(*weight, q, q.size(0), q.size(1))) return std::nullopt;
  for (const at::Tensor* t : {&q, &k, &v})
    if (reinterpret_cast<uintptr_t>(t->data_ptr()) & 15u) return std::nullopt;
  Call c{shape_of(q.sizes(), dtype, m, J, kappa, layout, flags), layout, status};
  if (fnb_check_shape(&c.shape)) return std::nullopt;
  py::gil_scoped_release nogil;
  c10::cuda::CUDAGuard guard(q.device());
  return run_attention(q, k, v, weight, c);
}

// The module's forward: projections, attention, output projection.  The caller has seen to it that the projections are plain
// bias-free linears without hooks.
std::optional<at::Tensor> module_forward(const at::Tensor& x, const at::Tensor& wq, const at::Tensor& wk, const at::Tensor& wv, const at::Tensor& wo,
                                         int64_t H, int64_t m, int64_t J, double kappa, const std::optional<at::Tensor>& conv,
                                         const at::Tensor& status) {
  if (c10::impl::dispatch_mode_enabled() || at::autocast::is_autocast_enabled(at::kCUDA)) return std::nullopt;
  const int64_t dim = x.dim() == 3 ? x.size(2) : 0;
  for (const at::Tensor* t : {&x, &wq, &wk, &wv, &wo})
    if (!plain(*t) || t->scalar_type() != x.scalar_type() || t->device() != x.device() || !t->is_contiguous() || has_tangent(*t)) return std::nullopt;
  for (const at::Tensor* t : {&wq, &wk, &wv, &wo})
    if (t->dim() != 2 || t->size(0) != dim || t->size(1) != dim) return std::nullopt;
  const uint32_t flags = g_flags.load();
  if (dim == 0 || x.numel() == 0 || H < 1 || dim % H || dtype_of(x) < 0 || !takes_numbers(m, J, kappa) || !takes_bnhd(dtype_of(x), dim / H, m, flags))
    return std::nullopt;
  if (status.device() != x.device() || (conv && !takes_taps(*conv, x, x.size(0), H))) return std::nullopt;
  const int64_t B = x.size(0), N = x.size(1);
  const int layout = H == 1 || N == 1 ? FNB_LAYOUT_BHND : FNB_LAYOUT_BNHD;      // (head-split views of one head or row are contiguous)
  const Call c{shape_of({B, H, N, dim / H}, dtype_of(x), m, J, kappa, layout, flags), layout, status};
  if (fnb_check_shape(&c.shape)) return std::nullopt;      // (refused further on; nothing has been formed yet)
  py::gil_scoped_release nogil;
  c10::cuda::CUDAGuard guard(x.device());
  variable_list qkv;
  if (at::GradMode::is_enabled() && (x.requires_grad() || wq.requires_grad() || wk.requires_grad() || wv.requires_grad())) {
    qkv = ProjectionsNode::apply(x, wq, wk, wv, H);
  } else {
    at::AutoGradMode off(false);
    const at::Tensor x2 = x.view({B * N, dim});
    for (const at::Tensor* w : {&wq, &wk, &wv}) qkv.push_back(head_split(x2, *w, B, N, H));
  }
  const at::Tensor o = run_attention(qkv[0], qkv[1], qkv[2], conv, c);
  if (at::GradMode::is_enabled() && (o.requires_grad() || wo.requires_grad())) return OutputNode::apply(o, wo);
  return project_out(o, wo);
}

// ---- causal attention with a decay, layer norm ------------------------------------------------------------------
using OptTensor = std::optional<at::Tensor>;

void check_cuda(const at::Tensor& t, const char* name, const at::Tensor& like) {
  TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor (flashnystrom_b200 has no CPU path)");
  TORCH_CHECK(t.layout() == at::kStrided, name, " must be a strided tensor");
  TORCH_CHECK(t.device() == like.device(), name, " is on ", t.device(), ", the others on ", like.device());
}
// Results of a backward that is itself not differentiable: a second derivative raises instead of leaving a term out.  `of`: what the
// results depend on; the node that raises lies between them and these, so that no way to them goes past it.
variable_list once_differentiable(variable_list grads, const char* what, const variable_list& of) {
  if (!at::GradMode::is_enabled()) return grads;
  const size_t n = grads.size();
  for (const at::Tensor& t : of) grads.push_back(t);
  variable_list r = (*std::make_shared<torch::autograd::DelayedError>(std::string(what) + " has no second derivative", grads.size()))(std::move(grads));
  r.resize(n);
  return r;
}

// (B, H, N, D) rows that the kernels can read where they lie: last dimension contiguous, no dimension spread out of one element
at::Tensor rows_in_place(const at::Tensor& given) {
  const at::Tensor t = given.resolve_neg();
  bool fine = t.stride(3) == 1 || t.size(3) == 1;
  for (int i = 0; i < 3; ++i) fine = fine && (t.size(i) == 1 || t.stride(i) > 0);
  return fine ? t : t.contiguous();
}
fnb_rows rows_arg(const at::Tensor& t) { return {t.data_ptr(), t.stride(0), t.stride(1), t.stride(2)}; }
// uninitialised, in the order that t's heads and rows have in memory
at::Tensor empty_rows_like(const at::Tensor& t) { return empty_in(t, t.stride(1) < t.stride(2) ? FNB_LAYOUT_BNHD : FNB_LAYOUT_BHND); }

struct DecayArgs {
  at::Tensor q, k, v, log_decay, initial, seq_lens;      // (the last two may be undefined)
  double scale;
  at::Tensor status;
};
fnb_decay_shape decay_shape(const at::Tensor& q, double scale) {
  fnb_decay_shape s{};
  s.batch = q.size(0); s.heads = q.size(1); s.seq_len = q.size(2); s.head_dim = (int32_t)std::min<int64_t>(q.size(3), INT32_MAX);
  s.dtype = dtype_of(q); s.scale = (float)scale; s.flags = g_flags.load() & FNB_FLAG_FORCE_GENERIC;
  return s;
}
float* floats_or_null(const at::Tensor& t) { return t.defined() ? t.data_ptr<float>() : nullptr; }
const int32_t* lens_or_null(const at::Tensor& t) { return t.defined() ? t.data_ptr<int32_t>() : nullptr; }

void check_state(const at::Tensor& t, const char* name, const at::Tensor& q) {
  check_cuda(t, name, q);
  TORCH_CHECK(t.scalar_type() == at::kFloat, name, " must be float32, got ", t.scalar_type());
  TORCH_CHECK(t.sizes() == at::IntArrayRef({q.size(0), q.size(1), q.size(3), q.size(3)}), name, " must be (B, H, D, D), got ", t.sizes());
}
void check_log_decay(const at::Tensor& g, const at::Tensor& q) {
  check_cuda(g, "log_decay", q);
  TORCH_CHECK(g.scalar_type() == at::kFloat && g.dim() == 1 && g.size(0) == q.size(1), "log_decay must be a float32 tensor with one value a head (", q.size(1),
              "), got ", g.scalar_type(), " ", g.sizes());
  TORCH_CHECK(!(at::GradMode::is_enabled() && g.requires_grad()), "log_decay is a constant here: it has no gradient");
}
DecayArgs decay_args(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& log_decay, double scale, const OptTensor& initial,
                     const OptTensor& seq_lens, const at::Tensor& status) {
  TORCH_CHECK(q.is_cuda(), "q must be a CUDA tensor (flashnystrom_b200 has no CPU path)");
  TORCH_CHECK(q.dim() == 4 && k.dim() == 4 && v.dim() == 4, "q, k, v must be 4D (B, H, N, D)");
  check_cuda(q, "q", q);
  check_cuda(k, "k", q);
  check_cuda(v, "v", q);
  TORCH_CHECK(k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(), "q, k, v dtypes must match");
  TORCH_CHECK(k.sizes() == q.sizes() && v.sizes() == q.sizes(), "q, k, v shapes must match, got ", q.sizes(), ", ", k.sizes(), " and ", v.sizes());
  TORCH_CHECK(dtype_of(q) >= 0, "Supported dtypes: float32, float16, bfloat16");
  check_log_decay(log_decay, q);
  if (initial) check_state(*initial, "initial_state", q);
  if (seq_lens) {
    check_cuda(*seq_lens, "seq_lens", q);
    TORCH_CHECK(seq_lens->scalar_type() == at::kInt && seq_lens->dim() == 1 && seq_lens->size(0) == q.size(0),
                "seq_lens must be an int32 tensor with one length a sequence (", q.size(0), "), got ", seq_lens->scalar_type(), " ", seq_lens->sizes());
  }
  return {q, k, v, log_decay, initial ? *initial : at::Tensor(), seq_lens ? *seq_lens : at::Tensor(), scale, status};
}
// (memory that holds what the tensor says: no negative bit)
at::Tensor in_memory(const at::Tensor& t) { return t.resolve_neg().contiguous(); }
at::Tensor contiguous_or_none(const at::Tensor& t) { return t.defined() ? in_memory(t) : t; }

// out, the state behind the last row (undefined unless wanted), the states at the cuts
struct DecayResult { at::Tensor out, final, segments; };
// segment_floats: room for the states at the cuts, what they take where it is below zero
DecayResult run_decay_forward(const DecayArgs& c, bool want_state, int64_t segment_floats = -1) {
  const at::Tensor q = rows_in_place(c.q), k = rows_in_place(c.k), v = rows_in_place(c.v);
  const at::Tensor g = in_memory(c.log_decay), initial = contiguous_or_none(c.initial), lens = contiguous_or_none(c.seq_lens);
  fnb_decay_fwd_args a{};
  a.shape = decay_shape(q, c.scale);
  check(fnb_check_decay_shape(&a.shape));
  DecayResult r;
  const auto f32 = q.options().dtype(at::kFloat);
  r.out = empty_rows_like(q);
  if (want_state) r.final = at::empty({q.size(0), q.size(1), q.size(3), q.size(3)}, f32);
  const int64_t cuts = (int64_t)fnb_decay_segment_floats(&a.shape);
  TORCH_CHECK(segment_floats < 0 || segment_floats >= cuts, "room for ", segment_floats, " floats of states at the cuts, ", cuts, " are needed");
  r.segments = at::empty({segment_floats < 0 ? cuts : segment_floats}, f32);
  const at::Tensor ws = bytes(fnb_decay_workspace_bytes(&a.shape), q);
  a.q = rows_arg(q); a.k = rows_arg(k); a.v = rows_arg(v); a.out = rows_arg(r.out);
  a.log_decay = g.data_ptr<float>(); a.seq_lens = lens_or_null(lens);
  a.initial_state = floats_or_null(initial); a.final_state = floats_or_null(r.final);
  a.segment_states = r.segments.numel() ? r.segments.data_ptr<float>() : nullptr;
  a.workspace = ws.data_ptr(); a.workspace_bytes = (size_t)ws.numel();
  a.device = q.device().index();
  a.stream = c10::cuda::getCurrentCUDAStream(q.device().index()).stream();
  a.device_status = c.status.data_ptr<int32_t>();
  check(fnb_decay_forward(&a));
  return r;
}
// dq, dk, dv, d_initial (undefined unless wanted)
variable_list run_decay_backward(const DecayArgs& c, const at::Tensor& segments, const at::Tensor& d_out, const at::Tensor& d_final, bool want_initial) {
  const at::Tensor q = rows_in_place(c.q), k = rows_in_place(c.k), v = rows_in_place(c.v), d = rows_in_place(d_out);
  const at::Tensor g = in_memory(c.log_decay), initial = contiguous_or_none(c.initial), lens = contiguous_or_none(c.seq_lens),
                   df = contiguous_or_none(d_final);
  fnb_decay_bwd_args a{};
  a.shape = decay_shape(q, c.scale);
  check(fnb_check_decay_shape(&a.shape));
  TORCH_CHECK(segments.scalar_type() == at::kFloat && segments.device() == q.device() && segments.is_contiguous() &&
                  segments.numel() >= (int64_t)fnb_decay_segment_floats(&a.shape),
              "the saved states do not match q");
  at::Tensor dq = empty_rows_like(q), dk = empty_rows_like(k), dv = empty_rows_like(v), d_initial;
  if (want_initial) d_initial = at::empty({q.size(0), q.size(1), q.size(3), q.size(3)}, q.options().dtype(at::kFloat));
  const at::Tensor ws = bytes(fnb_decay_workspace_bytes(&a.shape), q);
  a.q = rows_arg(q); a.k = rows_arg(k); a.v = rows_arg(v); a.d_out = rows_arg(d);
  a.dq = rows_arg(dq); a.dk = rows_arg(dk); a.dv = rows_arg(dv);
  a.log_decay = g.data_ptr<float>(); a.seq_lens = lens_or_null(lens); a.initial_state = floats_or_null(initial);
  a.d_final_state = floats_or_null(df); a.d_initial_state = floats_or_null(d_initial);
  a.segment_states = segments.numel() ? segments.data_ptr<float>() : nullptr;
  a.workspace = ws.data_ptr(); a.workspace_bytes = (size_t)ws.numel();
  a.device = q.device().index();
  a.stream = c10::cuda::getCurrentCUDAStream(q.device().index()).stream();
  a.device_status = c.status.data_ptr<int32_t>();
  check(fnb_decay_backward(&a));
  return {dq, dk, dv, d_initial};
}

struct DecayNode : torch::autograd::Function<DecayNode> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const OptTensor& initial,
                               const DecayArgs& c, bool want_state) {
    const at::Tensor s0 = initial ? *initial : at::Tensor();
    const DecayResult r = run_decay_forward({q, k, v, c.log_decay, s0, c.seq_lens, c.scale, c.status}, want_state);
    ctx->save_for_backward({q, k, v, s0, c.log_decay, c.seq_lens, r.segments});
    ctx->saved_data["scale"] = c.scale;
    ctx->saved_data["status"] = c.status;
    ctx->set_materialize_grads(false);
    if (want_state) return {r.out, r.final};
    return {r.out};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list kept = ctx->get_saved_variables();
    const DecayArgs c{kept[0], kept[1], kept[2], kept[4], kept[3], kept[5], ctx->saved_data["scale"].toDouble(), ctx->saved_data["status"].toTensor()};
    c10::cuda::CUDAGuard guard(c.q.device());
    at::Tensor d = grads[0], df = grads.size() > 1 ? grads[1] : at::Tensor();
    variable_list result(6);
    if (!d.defined() && !df.defined()) return result;
    if (!d.defined()) d = at::zeros_like(c.q);
    TORCH_CHECK(d.is_cuda() && d.device() == c.q.device() && d.sizes() == c.q.sizes() && d.scalar_type() == c.q.scalar_type(),
                "the gradient of the output does not match q in shape, dtype or device");
    if (df.defined()) check_state(df, "the gradient of the state", c.q);
    variable_list g;
    {
      at::AutoGradMode off(false);
      g = run_decay_backward(c, kept[6], d, df, c.initial.defined() && ctx->needs_input_grad(3));
    }
    for (int i = 0; i < 4; ++i)
      if (g[i].defined() && ctx->needs_input_grad(i)) result[i] = g[i];
    return once_differentiable(std::move(result), "decay_attention", {c.q, c.k, c.v, c.initial, d, df});
  }
};

// the state behind a sequence without rows
at::Tensor state_of_nothing(const DecayArgs& c) {
  TORCH_CHECK(c.q.size(3) > 0, "head_dim must be 16, 32, 64 or 128, got 0");
  return c.initial.defined() ? c.initial.clone() : at::zeros({c.q.size(0), c.q.size(1), c.q.size(3), c.q.size(3)}, c.q.options().dtype(at::kFloat));
}

// A subclass that does its own work on operators: the calls below return nothing for one, and the caller goes through the registered operators.
bool own_dispatch(const at::Tensor& t) { return at::isTensorSubclassLike(t); }
bool own_dispatch(const OptTensor& t) { return t && at::isTensorSubclassLike(*t); }
template <class... Ts> bool any_own_dispatch(const Ts&... t) { return (own_dispatch(t) || ...); }

// (out, final state or nothing)
std::optional<std::pair<at::Tensor, OptTensor>> decay_attention(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& log_decay,
                                                 double scale, const OptTensor& initial, const OptTensor& seq_lens, bool want_state,
                                                 const at::Tensor& status) {
  if (any_own_dispatch(q, k, v, log_decay, initial, seq_lens)) return std::nullopt;
  const DecayArgs c = decay_args(q, k, v, log_decay, scale, initial, seq_lens, status);
  py::gil_scoped_release nogil;
  c10::cuda::CUDAGuard guard(q.device());
  if (q.numel() == 0) {      // nothing to attend to: the state goes through
    OptTensor state = state_of_nothing(c);
    if (!want_state) state = std::nullopt;
    return std::make_pair(q + k + v, state);      // (no elements, and a graph to all three)
  }
  if (at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad() || (initial && initial->requires_grad()))) {
    const variable_list r = DecayNode::apply(q, k, v, initial, c, want_state);
    return std::make_pair(r[0], want_state ? OptTensor(r[1]) : std::nullopt);
  }
  at::AutoGradMode off(false);
  const DecayResult r = run_decay_forward(c, want_state);
  return std::make_pair(r.out, want_state ? OptTensor(r.final) : std::nullopt);
}
// For the registered operators: every result a tensor, without elements where it is not wanted.
at::Tensor or_nothing(const at::Tensor& t, const at::Tensor& like) { return t.defined() ? t : at::empty({0}, like.options()); }
std::tuple<at::Tensor, at::Tensor, at::Tensor> decay_forward(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& log_decay,
                                                             double scale, const OptTensor& initial, const OptTensor& seq_lens, bool want_state,
                                                             int64_t segment_floats, const at::Tensor& status) {
  at::AutoGradMode off(false);
  const DecayArgs c = decay_args(q, k, v, log_decay, scale, initial, seq_lens, status);
  c10::cuda::CUDAGuard guard(q.device());
  if (q.numel() == 0)
    return {empty_rows_like(rows_in_place(q)), or_nothing(want_state ? state_of_nothing(c) : at::Tensor(), log_decay), at::empty({std::max<int64_t>(segment_floats, 0)}, log_decay.options())};
  const DecayResult r = run_decay_forward(c, want_state, segment_floats);
  return {r.out, or_nothing(r.final, log_decay), r.segments};
}
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> decay_backward(const at::Tensor& d, const OptTensor& df, const at::Tensor& q,
                                                                          const at::Tensor& k, const at::Tensor& v, const at::Tensor& log_decay,
                                                                          double scale, const OptTensor& initial, const OptTensor& seq_lens,
                                                                          const at::Tensor& segments, bool want_initial, const at::Tensor& status) {
  at::AutoGradMode off(false);
  const DecayArgs c = decay_args(q, k, v, log_decay, scale, initial, seq_lens, status);
  TORCH_CHECK(d.sizes() == q.sizes() && d.scalar_type() == q.scalar_type() && d.device() == q.device(), "d_out does not match q");
  if (df) check_state(*df, "d_final_state", q);
  c10::cuda::CUDAGuard guard(q.device());
  if (q.numel() == 0) {
    const at::Tensor ds = !want_initial ? at::Tensor() : df ? df->clone() : at::zeros({q.size(0), q.size(1), q.size(3), q.size(3)}, log_decay.options());
    return {empty_rows_like(rows_in_place(q)), empty_rows_like(rows_in_place(k)), empty_rows_like(rows_in_place(v)), or_nothing(ds, log_decay)};
  }
  const variable_list g = run_decay_backward(c, segments, d, df ? *df : at::Tensor(), want_initial);
  return {g[0], g[1], g[2], or_nothing(g[3], log_decay)};
}

std::optional<at::Tensor> decay_step(const at::Tensor& q_, const at::Tensor& k_, const at::Tensor& v_, const at::Tensor& state, const at::Tensor& log_decay,
                      double scale, const OptTensor& slots) {
  if (any_own_dispatch(q_, k_, v_, state, log_decay, slots)) return std::nullopt;
  TORCH_CHECK(q_.is_cuda(), "q must be a CUDA tensor (flashnystrom_b200 has no CPU path)");
  TORCH_CHECK(q_.dim() == 3 && k_.dim() == 3 && v_.dim() == 3, "q, k, v must be 3D (B, H, D)");
  check_cuda(q_, "q", q_);
  check_cuda(k_, "k", q_);
  check_cuda(v_, "v", q_);
  check_cuda(state, "state", q_);
  TORCH_CHECK(k_.scalar_type() == q_.scalar_type() && v_.scalar_type() == q_.scalar_type(), "q, k, v dtypes must match");
  TORCH_CHECK(k_.sizes() == q_.sizes() && v_.sizes() == q_.sizes(), "q, k, v shapes must match");
  TORCH_CHECK(dtype_of(q_) >= 0, "Supported dtypes: float32, float16, bfloat16");
  check_log_decay(log_decay, q_);
  const int64_t B = q_.size(0), H = q_.size(1), D = q_.size(2);
  TORCH_CHECK(state.scalar_type() == at::kFloat && state.dim() == 4 && state.size(1) == H && state.size(2) == D && state.size(3) == D && state.is_contiguous(),
              "state must be a contiguous float32 tensor of shape (states, ", H, ", ", D, ", ", D, "), got ", state.scalar_type(), " ", state.sizes());
  TORCH_CHECK(slots || state.size(0) == B, "state must have one entry for each row (", B, ") where no slots are given, got ", state.size(0));
  if (slots) {
    check_cuda(*slots, "slots", q_);
    TORCH_CHECK(slots->scalar_type() == at::kInt && slots->dim() == 1 && slots->size(0) == B, "slots must be an int32 tensor with one value a row (", B, "), got ",
                slots->scalar_type(), " ", slots->sizes());
  }
  TORCH_CHECK(!(at::GradMode::is_enabled() && (q_.requires_grad() || k_.requires_grad() || v_.requires_grad() || state.requires_grad())),
              "decay_attention_step updates the state in place and has no gradient: use decay_attention, or torch.no_grad()");
  TORCH_CHECK(!state.is_neg(), "state must not be a negative view: it is written where it lies");
  TORCH_CHECK(!state.is_inference() || c10::InferenceMode::is_enabled(), "an inference tensor cannot be updated in place outside InferenceMode");
  py::gil_scoped_release nogil;
  c10::cuda::CUDAGuard guard(q_.device());
  at::AutoGradMode off(false);
  const auto in_place = [](const at::Tensor& t) { return t.stride(2) == 1 ? t.resolve_neg() : in_memory(t); };
  const at::Tensor q = in_place(q_), k = in_place(k_), v = in_place(v_), g = in_memory(log_decay);
  at::Tensor out = at::empty({B, H, D}, q.options());
  if (B == 0 || H == 0) return out;
  if (state.size(0) == 0) return out.zero_();      // (slots of no state: every row is idle)
  const at::Tensor s = slots ? in_memory(*slots) : at::Tensor();
  fnb_decay_step_args a{};
  const auto arg = [](const at::Tensor& t) { return fnb_rows{t.data_ptr(), t.stride(0), t.stride(1), 0}; };
  a.batch = B; a.heads = H; a.num_states = state.size(0); a.head_dim = (int32_t)std::min<int64_t>(D, INT32_MAX); a.dtype = dtype_of(q);
  a.scale = (float)scale;
  a.q = arg(q); a.k = arg(k); a.v = arg(v); a.out = arg(out);
  a.log_decay = g.data_ptr<float>(); a.states = state.data_ptr<float>(); a.slots = lens_or_null(s);
  a.device = q.device().index();
  a.stream = c10::cuda::getCurrentCUDAStream(q.device().index()).stream();
  check(fnb_decay_step(&a));
  if (!state.is_inference()) state.unsafeGetTensorImpl()->bump_version();
  return out;
}

// x as rows of its last dimension that lie one stride apart; contiguous where it is not so
at::Tensor norm_rows(const at::Tensor& given) {
  const at::Tensor x = given.resolve_neg();
  const int64_t C = x.size(-1);
  if (C == 1 || x.stride(-1) == 1) {
    int64_t stride = -1, size = 1;      // of the innermost leading dimension that counts; rows so far
    bool fine = true;
    for (int64_t i = x.dim() - 2; i >= 0 && fine; --i) {
      if (x.size(i) == 1) continue;
      if (stride < 0) stride = x.stride(i);
      else fine = x.stride(i) == size * stride;
      size *= x.size(i);
    }
    if (fine && (stride < 0 || stride >= C)) return x.as_strided({size, C}, {stride < 0 ? C : stride, 1});
  }
  return x.contiguous().view({-1, C});
}
struct NormArgs {
  at::Tensor x, weight, bias;      // (weight and bias may be undefined)
  int64_t groups;
  double eps;
};
fnb_norm_shape norm_shape(const at::Tensor& x, at::ScalarType param, int64_t groups, double eps) {
  fnb_norm_shape s{};
  TORCH_CHECK(x.size(-1) <= INT32_MAX, "the last dimension is too large (", x.size(-1), ")");
  s.rows = x.numel() / x.size(-1); s.cols = (int32_t)x.size(-1); s.groups = (int32_t)groups;
  s.dtype = dtype_of(x); s.param_dtype = param == at::kFloat ? FNB_F32 : s.dtype; s.eps = (float)eps;
  return s;
}
at::ScalarType norm_param_type(const NormArgs& c) {
  return c.weight.defined() ? c.weight.scalar_type() : c.bias.defined() ? c.bias.scalar_type() : at::kFloat;
}
NormArgs norm_args(const at::Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps, int64_t groups) {
  TORCH_CHECK(x.is_cuda(), "x must be a CUDA tensor (flashnystrom_b200 has no CPU path)");
  check_cuda(x, "x", x);
  TORCH_CHECK(dtype_of(x) >= 0, "Supported dtypes: float32, float16, bfloat16");
  TORCH_CHECK(x.dim() >= 1 && x.size(-1) > 0, "x must have a last dimension to normalise, got ", x.sizes());
  TORCH_CHECK(groups >= 1 && x.size(-1) % groups == 0, "num_groups (", groups, ") must divide the last dimension (", x.size(-1), ")");
  const struct { const OptTensor& t; const char* name; } params[] = {{weight, "weight"}, {bias, "bias"}};
  for (const auto& p : params)
    if (p.t) {
      check_cuda(*p.t, p.name, x);
      TORCH_CHECK(p.t->dim() == 1 && p.t->size(0) == x.size(-1), p.name, " must have ", x.size(-1), " values, got ", p.t->sizes());
      TORCH_CHECK(p.t->scalar_type() == x.scalar_type() || p.t->scalar_type() == at::kFloat, p.name, " must be float32 or ", x.scalar_type(), ", got ",
                  p.t->scalar_type());
    }
  TORCH_CHECK(!(weight && bias) || weight->scalar_type() == bias->scalar_type(), "weight and bias dtypes must match");
  return {x, weight ? *weight : at::Tensor(), bias ? *bias : at::Tensor(), groups, eps};
}
const void* data_or_null(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

struct NormResult { at::Tensor y, mean, rstd; };
NormResult run_norm_forward(const NormArgs& c, bool keep, bool apart = false) {      // apart: statistics in memory of their own each
  NormResult r;
  fnb_norm_fwd_args a{};
  a.shape = norm_shape(c.x, norm_param_type(c), c.groups, c.eps);
  const at::Tensor x = norm_rows(c.x), w = contiguous_or_none(c.weight), b = contiguous_or_none(c.bias);
  r.y = at::empty(c.x.sizes(), c.x.options());
  if (keep && apart) {
    r.mean = at::empty({a.shape.rows * c.groups}, c.x.options().dtype(at::kFloat));
    r.rstd = at::empty_like(r.mean);
  } else if (keep) {
    const at::Tensor stats = at::empty({2, a.shape.rows * c.groups}, c.x.options().dtype(at::kFloat));
    r.mean = stats.select(0, 0);
    r.rstd = stats.select(0, 1);
  }
  a.x = x.data_ptr(); a.x_stride = x.stride(0); a.y = r.y.data_ptr(); a.y_stride = x.size(1);
  a.weight = data_or_null(w); a.bias = data_or_null(b); a.mean = floats_or_null(r.mean); a.rstd = floats_or_null(r.rstd);
  a.device = x.device().index();
  a.stream = c10::cuda::getCurrentCUDAStream(x.device().index()).stream();
  check(fnb_norm_forward(&a));
  return r;
}
// d_x, d_weight, d_bias, those that are wanted
variable_list run_norm_backward(const at::Tensor& x_, const at::Tensor& weight, const at::Tensor& mean, const at::Tensor& rstd, const at::Tensor& d_,
                                int64_t groups, double eps, at::ScalarType param, bool want_x, bool want_w, bool want_b) {
  fnb_norm_bwd_args a{};
  a.shape = norm_shape(x_, param, groups, eps);
  check(fnb_check_norm_shape(&a.shape));
  const at::Tensor x = norm_rows(x_), d = norm_rows(d_), w = contiguous_or_none(weight);
  TORCH_CHECK(mean.is_contiguous() && rstd.is_contiguous() && mean.scalar_type() == at::kFloat && rstd.scalar_type() == at::kFloat && mean.device() == x.device() &&
                  rstd.device() == x.device() && mean.numel() == a.shape.rows * groups && rstd.numel() == a.shape.rows * groups,
              "the saved statistics do not match x");
  at::Tensor dx, dw, db, ws;
  if (want_x) dx = at::empty(x_.sizes(), x_.options());
  const auto po = x_.options().dtype(param);
  if (want_w) dw = at::empty({x.size(1)}, po);
  if (want_b) db = at::empty({x.size(1)}, po);
  if (want_w || want_b) {
    ws = bytes(fnb_norm_workspace_bytes(&a.shape), x);
    a.workspace = ws.data_ptr();
    a.workspace_bytes = (size_t)ws.numel();
  }
  a.x = x.data_ptr(); a.x_stride = x.stride(0); a.d_y = d.data_ptr(); a.d_y_stride = d.stride(0);
  a.d_x = want_x ? dx.data_ptr() : nullptr; a.d_x_stride = x.size(1); a.weight = data_or_null(w);
  a.mean = mean.data_ptr<float>(); a.rstd = rstd.data_ptr<float>();
  a.d_weight = want_w ? dw.data_ptr() : nullptr; a.d_bias = want_b ? db.data_ptr() : nullptr;
  a.device = x.device().index();
  a.stream = c10::cuda::getCurrentCUDAStream(x.device().index()).stream();
  check(fnb_norm_backward(&a));
  return {dx, dw, db};
}

struct NormNode : torch::autograd::Function<NormNode> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const OptTensor& weight, const OptTensor& bias, int64_t groups, double eps) {
    const NormArgs c{x, weight ? *weight : at::Tensor(), bias ? *bias : at::Tensor(), groups, eps};
    const NormResult r = run_norm_forward(c, true);
    ctx->save_for_backward({x, c.weight, r.mean, r.rstd});
    ctx->saved_data["bias"] = bias.has_value();
    ctx->saved_data["groups"] = groups;
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["param"] = (int64_t)norm_param_type(c);
    return r.y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list kept = ctx->get_saved_variables();
    const at::Tensor &x = kept[0], &d = grads[0];
    c10::cuda::CUDAGuard guard(x.device());
    TORCH_CHECK(d.is_cuda() && d.device() == x.device() && d.sizes() == x.sizes() && d.scalar_type() == x.scalar_type(),
                "the gradient of the output does not match x in shape, dtype or device");
    const bool has_w = kept[1].defined(), has_b = ctx->saved_data["bias"].toBool();      // (what is not given has no place among the inputs)
    variable_list g;
    {
      at::AutoGradMode off(false);
      g = run_norm_backward(x, kept[1], kept[2], kept[3], d, ctx->saved_data["groups"].toInt(), ctx->saved_data["eps"].toDouble(),
                            (at::ScalarType)ctx->saved_data["param"].toInt(), ctx->needs_input_grad(0), has_w && ctx->needs_input_grad(1),
                            has_b && ctx->needs_input_grad(has_w ? 2 : 1));
    }
    g.resize(5);
    return once_differentiable(std::move(g), "layer_norm", {x, kept[1], d});
  }
};
std::optional<at::Tensor> layer_norm(const at::Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps, int64_t groups) {
  if (any_own_dispatch(x, weight, bias)) return std::nullopt;
  const NormArgs c = norm_args(x, weight, bias, eps, groups);
  py::gil_scoped_release nogil;
  c10::cuda::CUDAGuard guard(x.device());
  if (x.numel() == 0) {      // no rows: gradients of weight and bias are zeros
    at::Tensor y = x.clone();
    if (weight) y = y * weight->to(x.scalar_type());
    return bias ? y + bias->to(x.scalar_type()) : y;
  }
  if (at::GradMode::is_enabled() && (x.requires_grad() || (weight && weight->requires_grad()) || (bias && bias->requires_grad())))
    return NormNode::apply(x, weight, bias, groups, eps);
  at::AutoGradMode off(false);
  return run_norm_forward(c, false).y;
}
std::tuple<at::Tensor, at::Tensor, at::Tensor> norm_forward(const at::Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps, int64_t groups,
                                                            bool keep) {
  at::AutoGradMode off(false);
  c10::cuda::CUDAGuard guard(x.device());
  const NormArgs c = norm_args(x, weight, bias, eps, groups);
  const at::Tensor none = at::empty({0}, x.options().dtype(at::kFloat));
  if (x.numel() == 0) return {at::empty(x.sizes(), x.options()), none, at::empty_like(none)};
  const NormResult r = run_norm_forward(c, keep, true);
  return {r.y, or_nothing(r.mean, none), or_nothing(r.rstd, none)};
}
std::tuple<at::Tensor, at::Tensor, at::Tensor> norm_backward(const at::Tensor& d, const at::Tensor& x, const OptTensor& weight, const at::Tensor& mean,
                                                             const at::Tensor& rstd, double eps, int64_t groups, bool param_f32, bool want_x, bool want_w,
                                                             bool want_b) {
  at::AutoGradMode off(false);
  c10::cuda::CUDAGuard guard(x.device());
  norm_args(x, weight, std::nullopt, eps, groups);
  TORCH_CHECK(d.sizes() == x.sizes() && d.scalar_type() == x.scalar_type() && d.device() == x.device(), "d_y does not match x");
  const at::ScalarType param = param_f32 ? at::kFloat : x.scalar_type();
  const at::Tensor none = at::empty({0}, x.options().dtype(param));
  if (x.numel() == 0) {
    const auto zeros = [&](bool want) { return want ? at::zeros({x.size(-1)}, none.options()) : at::empty_like(none); };
    return {want_x ? at::empty(x.sizes(), x.options()) : at::empty({0}, x.options()), zeros(want_w), zeros(want_b)};
  }
  const variable_list g = run_norm_backward(x, weight ? *weight : at::Tensor(), mean, rstd, d, groups, eps, param, want_x, want_w, want_b);
  return {or_nothing(g[0], x), or_nothing(g[1], none), or_nothing(g[2], none)};
}

}  // namespace

PYBIND11_MODULE(_native, mod) {
  mod.def("attention", &attention);
  mod.def("module_forward", &module_forward);
  mod.def("decay_attention", &decay_attention);
  mod.def("decay_forward", &decay_forward);
  mod.def("decay_backward", &decay_backward);
  mod.def("decay_step", &decay_step);
  mod.def("layer_norm", &layer_norm);
  mod.def("norm_forward", &norm_forward);
  mod.def("norm_backward", &norm_backward);
  mod.def("set_flags", [](uint32_t flags) { g_flags = flags; });
  mod.def("set_debug", [](py::object f) { g_debug = f.release().ptr(); });
}
