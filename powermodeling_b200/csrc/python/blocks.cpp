// _blocksnative: the block operators on torch tensors (host C++ over the C
// entries of include/pmb200_blocks.h).
//
// A call of a few microseconds on the GPU must not wait for Python to read
// shapes and strides one by one, so the checks, the output allocations and
// the job structs of powermodeling_b200/blocks.py are here.  A refused
// argument raises ValueError, a failed native call the package's NativeError.
// Work goes to the current stream of the tensors' device; nothing else is
// synchronized, kept or allocated but the outputs and a scratch tensor, which
// the caching allocator hands back in that stream's order.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/Functions.h>
#include <ATen/MemoryOverlap.h>
#include <ATen/TracerMode.h>
#include <ATen/core/Tensor.h>
#include <c10/core/GradMode.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/variable.h>

#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <optional>
#include <string>

#include "pmb200.h"
#include "pmb200_blocks.h"

namespace {

PyObject* g_native_error = nullptr;

struct Refused {
  std::string message;
};
struct NativeFailure {
  std::string message;
};

[[noreturn]] void refuse(const char* fmt, ...) {
  char text[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(text, sizeof text, fmt, ap);
  va_end(ap);
  throw Refused{text};
}

void check(int rc, const char* what) {
  if (rc == PM_OK) return;
  char text[1024];
  pm_last_error(text, sizeof text);
  throw NativeFailure{std::string(what) + " failed (" + std::to_string(rc) + "): " + text};
}

// The calls read memory by themselves, past torch's dispatcher: tensors whose values are not what lies there, or that
// stand for others, and whatever records or follows the dispatcher's calls would be answered wrongly without an error.
const at::Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) refuse("%s must be a tensor", name);
  const at::Tensor& t = THPVariable_Unpack(o);
  constexpr c10::DispatchKeySet kNotPlain({c10::DispatchKey::Python, c10::DispatchKey::FuncTorchBatched, c10::DispatchKey::FuncTorchGradWrapper,
                                           c10::DispatchKey::Functionalize, c10::DispatchKey::Negative, c10::DispatchKey::Conjugate,
                                           c10::DispatchKey::ZeroTensor});
  if (t.layout() != at::kStrided || t.key_set().has_any(kNotPlain))
    refuse("%s must be a plain strided tensor (not one of vmap, functorch or a dispatch subclass, nor lazily negated)", name);
  if (t._fw_grad(0).defined()) refuse("%s has a forward-mode tangent, and the block operators have no forward-mode gradient", name);
  return t;
}
void not_recorded() {
  using c10::impl::TorchDispatchModeKey;
  bool recorded = at::tracer::impl::is_dispatch_enabled();
  if (c10::impl::TorchDispatchModeTLS::any_modes_set())
    for (const TorchDispatchModeKey k : {TorchDispatchModeKey::FAKE, TorchDispatchModeKey::PROXY, TorchDispatchModeKey::FUNCTIONAL})
      recorded = recorded || c10::impl::TorchDispatchModeTLS::get_mode(k).has_value();
  if (recorded) refuse("the block operators cannot be traced: call them outside torch.jit.trace, make_fx and fake tensors' modes");
}
// The tensor, or an undefined one for None.
at::Tensor maybe(PyObject* o, const char* name) { return o == Py_None ? at::Tensor() : tensor(o, name); }

double number(PyObject* o) {
  if (THPVariable_Check(o) && THPVariable_Unpack(o).requires_grad()) refuse("scale and eps are numbers: no gradient goes through them");
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw python_error();
  return v;
}
int64_t integer(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw python_error();
  return v;
}

int type_of(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return PM_DT_F32;
    case at::kBFloat16: return PM_DT_BF16;
    case at::kHalf: return PM_DT_F16;
    default: return -1;
  }
}

std::string shape_text(at::IntArrayRef s) {
  std::string t = "[";
  for (size_t i = 0; i < s.size(); ++i) t += (i ? ", " : "") + std::to_string(s[i]);
  return t + "]";
}

// Row stride of a 2-D tensor whose rows are contiguous and apart; one row has none, whatever the tensor says.
int64_t rows_of(const char* name, const at::Tensor& t) {
  if (t.dim() != 2) refuse("%s must be two-dimensional, got %s", name, shape_text(t.sizes()).c_str());
  if (t.size(1) > 1 && t.stride(1) != 1) refuse("%s: elements of a row must be contiguous", name);
  if (t.size(0) <= 1) return t.size(1);
  if (t.stride(0) < t.size(1)) refuse("%s: rows overlap", name);
  return t.stride(0);
}

// The one CUDA device of the tensors, made current for the call.
struct Place {
  c10::Device device{c10::kCPU};
  const char* who;
  Place(const char* who, std::initializer_list<const at::Tensor*> tensors) : who(who) {
    bool first = true;
    for (const at::Tensor* t : tensors) {
      if (!t->defined()) continue;
      if (first) device = t->device(), first = false;
      else if (t->device() != device)
        refuse("%s: tensors are on %s and %s", who, device.str().c_str(), t->device().str().c_str());
    }
    if (!device.is_cuda()) refuse("%s: tensors must be on a CUDA device", who);
  }
};

void* stream_of(const c10::Device& d) { return c10::cuda::getCurrentCUDAStream(d.index()).stream(); }
at::Tensor scratch_of(size_t bytes, const at::Tensor& like) {
  return at::empty({int64_t(bytes ? bytes : 1)}, like.options().dtype(at::kByte).requires_grad(false));
}
at::Tensor made(at::IntArrayRef shape, const at::Tensor& like) { return at::empty(shape, like.options().requires_grad(false)); }
at::Tensor made(at::IntArrayRef shape, const at::Tensor& like, at::ScalarType t) {
  return at::empty(shape, like.options().dtype(t).requires_grad(false));
}
void no_backward(const char* who, std::initializer_list<const at::Tensor*> tensors) {
  if (!c10::GradMode::is_enabled()) return;
  for (const at::Tensor* t : tensors)
    if (t->defined() && t->requires_grad()) refuse("%s has no backward: call it under torch.no_grad() or on detached tensors", who);
}
PyObject* wrap(const at::Tensor& t) {
  if (!t.defined()) Py_RETURN_NONE;
  return THPVariable_Wrap(t);
}

// ---------------------------------------------------------------- norms around a block
struct Norm {
  at::Tensor residual, block, pre, post, gate;
  pm_block_norm job{};
  // args: residual, block, pre_weight, post_weight, gate, scale
  explicit Norm(PyObject* const* args) {
    const char* who = "block_norm";
    residual = tensor(args[0], "residual");
    block = tensor(args[1], "block");
    pre = tensor(args[2], "pre_weight");
    post = maybe(args[3], "post_weight");
    gate = maybe(args[4], "gate");
    job.scale = float(number(args[5]));
    const at::ScalarType t = residual.scalar_type();
    if (type_of(t) < 0 || block.scalar_type() != t)
      refuse("%s: residual and block must share one of float32, bfloat16, float16", who);
    job.residual_stride = rows_of("residual", residual);
    job.block_stride = rows_of("block", block);
    if (block.sizes() != residual.sizes())
      refuse("block must be %s, got %s", shape_text(residual.sizes()).c_str(), shape_text(block.sizes()).c_str());
    job.rows = residual.size(0);
    const int64_t width = residual.size(1);
    if (width < 1 || width > (1 << 20)) refuse("%s: rows must not be empty or longer than 2^20", who);
    job.width = int32_t(width);
    job.dtype = type_of(t);
    auto weight = [&](const char* name, const at::Tensor& w) {
      if (w.dim() != 1 || w.size(0) != width || !w.is_contiguous() || (w.scalar_type() != t && w.scalar_type() != at::kFloat))
        refuse("%s: %s must be a contiguous [%lld] of the activations' type or float32", who, name, (long long)width);
      return type_of(w.scalar_type());
    };
    job.pre_dtype = weight("pre_weight", pre);
    if (post.defined()) job.post_dtype = weight("post_weight", post);
    if (gate.defined()) {
      const int64_t s = gate.dim() == 1 ? 1 : gate.dim() == 2 ? gate.size(0) : 0;
      if (s < 1 || gate.size(gate.dim() - 1) != width || !gate.is_contiguous() || job.rows % s ||
          (gate.scalar_type() != t && gate.scalar_type() != at::kFloat))
        refuse("%s: gate must be a contiguous [s, %lld] (s dividing %lld) of the activations' type or float32", who,
               (long long)width, (long long)job.rows);
      job.gate_rows = s;
      job.gate_dtype = type_of(gate.scalar_type());
    }
    if (!std::isfinite(job.scale)) refuse("%s: scale must be finite", who);
    job.residual = residual.const_data_ptr();
    job.block = block.const_data_ptr();
    job.pre_weight = pre.const_data_ptr();
    job.post_weight = post.defined() ? post.const_data_ptr() : nullptr;
    job.gate = gate.defined() ? gate.const_data_ptr() : nullptr;
  }
};

// block_norm(residual, block, pre_weight, post_weight, gate, scale, eps, want_stats) -> (hidden, normed[, stats])
PyObject* block_norm(PyObject* const* args) {
  Norm n(args);
  n.job.eps = float(number(args[6]));
  if (!(n.job.eps >= 0.0f) || !std::isfinite(n.job.eps)) refuse("block_norm: eps must be finite and >= 0");
  const bool want = PyObject_IsTrue(args[7]);
  const Place place("block_norm", {&n.residual, &n.block, &n.pre, &n.post, &n.gate});
  const c10::cuda::CUDAGuard guard(place.device);
  const at::Tensor hidden = made(n.residual.sizes(), n.residual), normed = made(n.residual.sizes(), n.residual);
  at::Tensor stats;
  if (want) stats = made({n.job.rows, 2}, n.residual, at::kFloat);
  if (n.job.rows) {
    n.job.hidden = hidden.mutable_data_ptr();
    n.job.normed = normed.mutable_data_ptr();
    n.job.stats = want ? stats.mutable_data_ptr<float>() : nullptr;
    check(pm_block_norm_device(&n.job, stream_of(place.device)), "pm_block_norm_device");
  }
  return want ? Py_BuildValue("(NNN)", wrap(hidden), wrap(normed), wrap(stats)) : Py_BuildValue("(NN)", wrap(hidden), wrap(normed));
}

// block_norm_backward(residual, block, pre_weight, post_weight, gate, scale, grad_hidden, grad_normed, stats,
//                     weight_grads, gate_grad) -> five tensors or None
PyObject* block_norm_backward(PyObject* const* args) {
  const char* who = "block_norm_backward";
  Norm n(args);
  const at::Tensor gh = maybe(args[6], "grad_hidden"), gy = maybe(args[7], "grad_normed"), stats = tensor(args[8], "stats");
  const bool weights = PyObject_IsTrue(args[9]), gates = PyObject_IsTrue(args[10]);
  if (stats.dim() != 2 || stats.size(0) != n.job.rows || stats.size(1) != 2 || stats.scalar_type() != at::kFloat || !stats.is_contiguous())
    refuse("%s: stats must be the forward call's [%lld, 2] float32", who, (long long)n.job.rows);
  if (!gh.defined() && !gy.defined()) refuse("%s: no incoming gradient", who);
  pm_block_norm_grads d{};
  auto incoming = [&](const char* name, const at::Tensor& g, int64_t* stride, const void** p) {
    if (!g.defined()) return;
    if (g.scalar_type() != n.residual.scalar_type()) refuse("%s: %s must be of the activations' type", who, name);
    *stride = rows_of(name, g);
    if (g.sizes() != n.residual.sizes()) refuse("%s must be %s", name, shape_text(n.residual.sizes()).c_str());
    *p = g.const_data_ptr();
  };
  incoming("grad_hidden", gh, &d.grad_hidden_stride, &d.grad_hidden);
  incoming("grad_normed", gy, &d.grad_normed_stride, &d.grad_normed);
  const Place place(who, {&n.residual, &n.block, &n.pre, &n.post, &n.gate, &gh, &gy, &stats});
  const c10::cuda::CUDAGuard guard(place.device);
  const at::Tensor gr = made(n.residual.sizes(), n.residual), gb = made(n.residual.sizes(), n.residual);
  at::Tensor gpre, gpost, ggate;
  if (weights) gpre = made(n.pre.sizes(), n.pre);
  if (weights && n.post.defined()) gpost = made(n.post.sizes(), n.post);
  if (gates && n.gate.defined()) ggate = made(n.gate.sizes(), n.gate);
  d.grad_residual = gr.mutable_data_ptr();
  d.grad_block = gb.mutable_data_ptr();
  d.grad_pre = gpre.defined() ? gpre.mutable_data_ptr() : nullptr;
  d.grad_post = gpost.defined() ? gpost.mutable_data_ptr() : nullptr;
  d.grad_gate = ggate.defined() ? ggate.mutable_data_ptr() : nullptr;
  n.job.stats = const_cast<float*>(stats.const_data_ptr<float>());
  const size_t need = pm_block_norm_backward_scratch_bytes(n.job.rows, n.job.gate_rows, n.job.width);
  const at::Tensor scratch = scratch_of(need, n.residual);
  check(pm_block_norm_backward_device(&n.job, &d, scratch.mutable_data_ptr(), need, stream_of(place.device)),
        "pm_block_norm_backward_device");
  return Py_BuildValue("(NNNNN)", wrap(gr), wrap(gb), wrap(gpre), wrap(gpost), wrap(ggate));
}

// ---------------------------------------------------------------- 4-bit weights
// matvec_w4(x, weight, scales, zeros, group_size) -> y
PyObject* matvec_w4(PyObject* const* args) {
  const char* who = "matvec_w4";
  const at::Tensor &x = tensor(args[0], "x"), &weight = tensor(args[1], "weight"), &scales = tensor(args[2], "scales");
  const at::Tensor zeros = maybe(args[3], "zeros");
  const int64_t group = integer(args[4]);
  const at::ScalarType t = x.scalar_type();
  if (t != at::kBFloat16 && t != at::kHalf) refuse("%s: x must be bfloat16 or float16", who);
  pm_matvec_w4 j{};
  j.x_stride = rows_of("x", x);
  const int64_t tokens = x.size(0), k = x.size(1);
  if (weight.scalar_type() != at::kByte || weight.dim() != 2 || !k || weight.size(1) != (k + 1) / 2)
    refuse("%s: weight must be uint8 [n, %lld]", who, (long long)((k + 1) / 2));
  j.weight_stride = rows_of("weight", weight);
  if (j.weight_stride > (1 << 23) && weight.size(0) > 1) refuse("%s: weight rows lie at most 2^23 bytes apart", who);
  const int64_t n = weight.size(0);
  if (group < 32 || group % 32 || group > (1 << 24)) refuse("%s: group_size must be a multiple of 32", who);
  const int64_t groups = (k + group - 1) / group;
  if (scales.dim() != 2 || scales.size(0) != n || scales.size(1) != groups || !scales.is_contiguous() ||
      (scales.scalar_type() != t && scales.scalar_type() != at::kFloat))
    refuse("%s: scales must be a contiguous [%lld, %lld] of x's type or float32", who, (long long)n, (long long)groups);
  if (zeros.defined() && (zeros.dim() != 2 || zeros.size(0) != n || zeros.size(1) != groups || !zeros.is_contiguous() ||
                          zeros.scalar_type() != at::kByte))
    refuse("%s: zeros must be a contiguous [%lld, %lld] of uint8", who, (long long)n, (long long)groups);
  if (tokens > (1 << 16) || n > (1 << 24) || k > (1 << 24)) refuse("%s: at most 2^16 tokens, n and k at most 2^24", who);
  no_backward(who, {&x, &scales});
  const Place place(who, {&x, &weight, &scales, &zeros});
  const c10::cuda::CUDAGuard guard(place.device);
  const at::Tensor y = made({tokens, n}, x);
  if (y.numel()) {
    j.tokens = int32_t(tokens);
    j.n = int32_t(n);
    j.k = int32_t(k);
    j.group = int32_t(group);
    j.dtype = type_of(t);
    j.scales_dtype = type_of(scales.scalar_type());
    j.x = x.const_data_ptr();
    j.weight = static_cast<const uint8_t*>(weight.const_data_ptr());
    j.scales = scales.const_data_ptr();
    j.zeros = zeros.defined() ? static_cast<const uint8_t*>(zeros.const_data_ptr()) : nullptr;
    j.y = y.mutable_data_ptr();
    const size_t need = pm_matvec_w4_scratch_bytes(j.tokens, j.n, j.k);
    at::Tensor scratch;
    if (need) scratch = scratch_of(need, x);
    check(pm_matvec_w4_device(&j, need ? scratch.mutable_data_ptr() : nullptr, need, stream_of(place.device)), "pm_matvec_w4_device");
  }
  return wrap(y);
}

// ---------------------------------------------------------------- paged attention
// paged_attention(q, k_cache, v_cache, page_table, lengths, new_k, new_v, scale, window, layout, return_lse)
PyObject* paged_attention(PyObject* const* args) {
  const char* who = "paged_attention";
  const at::Tensor &q = tensor(args[0], "q"), &kc = tensor(args[1], "k_cache"), &vc = tensor(args[2], "v_cache"),
                   &table = tensor(args[3], "page_table"), &lengths = tensor(args[4], "lengths");
  const at::Tensor nk = maybe(args[5], "new_k"), nv = maybe(args[6], "new_v");
  const int64_t window = integer(args[8]);
  const char* layout = PyUnicode_Check(args[9]) ? PyUnicode_AsUTF8(args[9]) : "";
  const bool nhd = layout && std::string(layout) == "NHD", hnd = layout && std::string(layout) == "HND";
  const bool want_lse = PyObject_IsTrue(args[10]);
  const at::ScalarType t = q.scalar_type();
  if (t != at::kBFloat16 && t != at::kHalf) refuse("%s: q must be bfloat16 or float16", who);
  if (q.dim() != 3 || kc.dim() != 4 || (!nhd && !hnd))
    refuse("%s: q is [batch, q_heads, head_dim], a cache four-dimensional in layout NHD or HND", who);
  const int64_t batch = q.size(0), q_heads = q.size(1), head_dim = q.size(2);
  const int token = nhd ? 1 : 2, head = nhd ? 2 : 1;
  const int64_t pages = kc.size(0), page_size = kc.size(token), kv_heads = kc.size(head);
  if (!kv_heads || !q_heads || q_heads % kv_heads)
    refuse("%s: %lld key heads do not divide %lld query heads", who, (long long)kv_heads, (long long)q_heads);
  if (head_dim % 8 || head_dim < 8 || head_dim > 256) refuse("%s: head_dim must be a multiple of 8 up to 256", who);
  if (page_size < 1 || page_size > 65536 || window < 0 || window > INT32_MAX || pages > INT32_MAX)
    refuse("%s: page_size must be in 1..65536 and window >= 0", who);
  if (batch * q_heads > (1 << 24) || batch > (1 << 24)) refuse("%s: at most 2^24 query rows", who);
  if (kc.size(3) != head_dim) refuse("%s: k_cache holds heads of %lld elements, q of %lld", who, (long long)kc.size(3), (long long)head_dim);
  pm_paged_attention j{};
  // strides of the leading axes, 0 for an axis of one entry
  auto strided = [&](const char* name, const at::Tensor& a, at::IntArrayRef shape, int64_t* s) {
    if (a.sizes() != shape || a.scalar_type() != t) refuse("%s: %s must be %s of q's type", who, name, shape_text(shape).c_str());
    const int last = int(a.dim()) - 1;
    if (a.stride(last) != 1) refuse("%s: %s: the head's elements must be contiguous", who, name);
    bool ok = reinterpret_cast<uintptr_t>(a.const_data_ptr()) % 16 == 0;
    for (int i = 0; i < last; ++i) {
      s[i] = a.size(i) > 1 ? a.stride(i) : 0;
      ok = ok && s[i] % 8 == 0;
    }
    if (!ok) refuse("%s: %s must be 16-byte aligned with strides in multiples of 8 elements", who, name);
  };
  int64_t qs[2], ks[3], vs[3], nks[2] = {0, 0}, nvs[2] = {0, 0};
  strided("q", q, q.sizes(), qs);
  strided("k_cache", kc, kc.sizes(), ks);
  strided("v_cache", vc, kc.sizes(), vs);
  if (nk.defined() != nv.defined()) refuse("%s: new_k and new_v come together", who);
  if (nk.defined()) {
    const int64_t shape[3] = {batch, kv_heads, head_dim};
    strided("new_k", nk, shape, nks);
    strided("new_v", nv, shape, nvs);
    // written in place: every entry has to be its own
    if (at::has_internal_overlap(kc) == at::MemOverlap::Yes || at::has_internal_overlap(vc) == at::MemOverlap::Yes)
      refuse("%s: entries of the caches share memory, and the new token's would be written to all of them", who);
    if (at::get_overlap_status(kc, vc) == at::MemOverlapStatus::Full) refuse("%s: k_cache and v_cache are the same memory", who);
  }
  if (table.dim() != 2 || table.size(0) != batch || table.scalar_type() != at::kInt || (table.size(1) > 1 && table.stride(1) != 1) ||
      table.size(1) > INT32_MAX)
    refuse("%s: page_table must be int32 [%lld, columns] with contiguous rows", who, (long long)batch);
  if (lengths.dim() != 1 || lengths.size(0) != batch || lengths.scalar_type() != at::kInt || !lengths.is_contiguous())
    refuse("%s: lengths must be a contiguous int32 [%lld]", who, (long long)batch);
  j.scale = args[7] == Py_None ? float(1.0 / std::sqrt(double(head_dim))) : float(number(args[7]));
  if (!std::isfinite(j.scale)) refuse("%s: scale must be finite", who);
  no_backward(who, {&q, &kc, &vc, &nk, &nv});
  const Place place(who, {&q, &kc, &vc, &table, &lengths, &nk, &nv});
  const c10::cuda::CUDAGuard guard(place.device);
  const at::Tensor out = made({batch, q_heads, head_dim}, q);
  at::Tensor lse;
  if (want_lse) lse = made({batch, q_heads}, q, at::kFloat);
  if (batch) {
    j.batch = int32_t(batch);
    j.q_heads = int32_t(q_heads);
    j.kv_heads = int32_t(kv_heads);
    j.head_dim = int32_t(head_dim);
    j.page_size = int32_t(page_size);
    j.n_pages = int32_t(pages);
    j.table_columns = int32_t(table.size(1));
    j.dtype = type_of(t);
    j.window = int32_t(window);
    j.q_stride = qs[0], j.q_head_stride = qs[1];
    j.k_page_stride = ks[0], j.k_token_stride = ks[token], j.k_head_stride = ks[head];
    j.v_page_stride = vs[0], j.v_token_stride = vs[token], j.v_head_stride = vs[head];
    j.new_k_stride = nks[0], j.new_k_head_stride = nks[1];
    j.new_v_stride = nvs[0], j.new_v_head_stride = nvs[1];
    j.table_stride = table.stride(0);
    j.q = q.const_data_ptr();
    j.k_cache = const_cast<void*>(kc.const_data_ptr());
    j.v_cache = const_cast<void*>(vc.const_data_ptr());
    j.table = table.size(1) ? static_cast<const int32_t*>(table.const_data_ptr()) : nullptr;
    j.lengths = static_cast<const int32_t*>(lengths.const_data_ptr());
    j.new_k = nk.defined() ? nk.const_data_ptr() : nullptr;
    j.new_v = nv.defined() ? nv.const_data_ptr() : nullptr;
    j.out = out.mutable_data_ptr();
    j.lse = want_lse ? lse.mutable_data_ptr<float>() : nullptr;
    const size_t need = pm_paged_attention_scratch_bytes(j.batch, j.q_heads, j.kv_heads, j.head_dim);
    const at::Tensor scratch = scratch_of(need, q);
    check(pm_paged_attention_device(&j, scratch.mutable_data_ptr(), need, stream_of(place.device)), "pm_paged_attention_device");
    if (nk.defined()) {
      // autograd's count of in-place changes, where there is one
      if (!kc.is_inference()) kc.unsafeGetTensorImpl()->bump_version();
      if (!vc.is_inference()) vc.unsafeGetTensorImpl()->bump_version();
    }
  }
  if (!want_lse) return wrap(out);
  return Py_BuildValue("(NN)", wrap(out), wrap(lse));
}

// captured(tensor) -> whether the current stream of the tensor's device is being captured
PyObject* captured(PyObject* const* args) {
  const c10::Device device = tensor(args[0], "residual").device();
  if (!device.is_cuda()) Py_RETURN_FALSE;
  const c10::cuda::CUDAGuard guard(device);
  return PyBool_FromLong(c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None);
}

// held_outside_capture(residual, block, pre_weight, post_weight, gate) -> index of the first leaf whose gradient a living
// graph of the default stream accumulates, -1 without one.  The autograd engine would wait on that stream for a captured
// backward's gradients, which ends the capture.
PyObject* held_outside_capture(PyObject* const* args) {
  for (int i = 0; i < 5; ++i) {
    const at::Tensor t = maybe(args[i], "an input");
    if (!t.defined() || !t.is_cuda() || !t.requires_grad() || !t.is_leaf()) continue;
    const std::shared_ptr<torch::autograd::Node> node = torch::autograd::impl::try_get_grad_accumulator(t);
    if (!node) continue;
    const std::optional<c10::Stream> stream = node->stream();
    if (stream && *stream == c10::cuda::getDefaultCUDAStream(t.device().index()).unwrap()) return PyLong_FromLong(i);
  }
  return PyLong_FromLong(-1);
}

template <PyObject* (*Body)(PyObject* const*), int Count>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  if (count != Count) return PyErr_Format(PyExc_TypeError, "expected %d arguments, got %zd", Count, count);
  try {
    not_recorded();
    return Body(args);
  } catch (const Refused& r) {
    PyErr_SetString(PyExc_ValueError, r.message.c_str());
  } catch (const NativeFailure& f) {
    PyErr_SetString(g_native_error, f.message.c_str());
  }
  return nullptr;
  END_HANDLE_TH_ERRORS
}

template <PyObject* (*Body)(PyObject* const*), int Count>
constexpr PyMethodDef method(const char* name) {
  return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(&entry<Body, Count>)), METH_FASTCALL, nullptr};
}

PyMethodDef g_methods[] = {method<block_norm, 8>("block_norm"), method<block_norm_backward, 11>("block_norm_backward"),
                           method<matvec_w4, 5>("matvec_w4"), method<paged_attention, 11>("paged_attention"),
                           method<captured, 1>("captured"), method<held_outside_capture, 5>("held_outside_capture"), {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_blocksnative", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__blocksnative(void) {
  PyObject* native = PyImport_ImportModule("powermodeling_b200._native");
  if (!native) return nullptr;
  g_native_error = PyObject_GetAttrString(native, "NativeError");
  Py_DECREF(native);
  if (!g_native_error) return nullptr;
  return PyModule_Create(&g_module);
}
