// Python binding of libdlt_hip.so for torch tensors: argument checks, output allocation, the autograd nodes and the
// calls into the C ABI, compiled.  The Python modules next to it only name the entry points.
//
// A training step of one attention layer is three kernel launches of 10 ... 20 us each on the sizes most layers have.
// Through torch.autograd.Function and ctypes the host needed 146 us for that step (two Python frames per direction,
// descriptor and stride arrays built object by object, a device guard object, three to seven torch.empty calls from
// Python), so every such step waited for the host.  Here the same work is done on the tensor structs themselves.
//
// Nothing is kept from one call for the next and nothing is launched that the Python version did not launch.  The Python
// classes (torch.autograd.Function) stay the general path: a compiled entry point answers NotImplemented to every call that is
// not a plain eager one (see plain() below), and apply() of its class then goes on through the class.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/core/LegacyTypeDispatch.h>
#include <ATen/MemoryOverlap.h>
#include <ATen/hip/EmptyTensor.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/VariableTypeUtils.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/saved_variable.h>

#include <algorithm>
#include <array>
#include <mutex>
#include <string>
#include <vector>

#include "../../include/dlt.h"

namespace {

using at::Tensor;
using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

PyObject* g_dlt_error = nullptr;   // dl_templates_amd._lib.DltError

// ---- errors ---------------------------------------------------------------------------------
// Python exceptions that can also leave an engine thread: the error is kept inside the C++ exception.
[[noreturn]] void raise_py(PyObject* type, const std::string& msg) {
  pybind11::gil_scoped_acquire gil;
  PyErr_SetString(type, msg.c_str());
  python_error e;
  e.persist();
  throw std::move(e);
}

void require(bool ok, PyObject* type, const char* msg) {
  if (C10_UNLIKELY(!ok)) raise_py(type, msg);
}
void check_assert(bool ok, const char* msg) { require(ok, PyExc_AssertionError, msg); }

void check_rc(int rc) {
  if (C10_LIKELY(rc == DLT_OK)) return;
  const std::string msg = dlt_last_error();
  pybind11::gil_scoped_acquire gil;
  PyObject* exc = PyObject_CallFunction(g_dlt_error, "is", rc, msg.c_str());
  if (exc != nullptr) {
    PyErr_SetObject(g_dlt_error, exc);
    Py_DECREF(exc);
  }
  python_error e;
  e.persist();
  throw std::move(e);
}

std::string shown(const at::Device& d) { return d.str(); }

// every tensor on one ROCm device
template <typename... T>
void require_gpu(const Tensor& first, const T&... rest) {
  const at::Device dev = first.device();
  auto one = [&](const Tensor& t) {
    if (C10_UNLIKELY(!t.is_cuda()))
      raise_py(PyExc_RuntimeError, "dl_templates_amd runs on a ROCm GPU only: got a tensor on " + shown(t.device()));
    if (C10_UNLIKELY(t.device() != dev))
      raise_py(PyExc_RuntimeError, "all tensors must be on one device, got " + shown(dev) + " and " + shown(t.device()));
  };
  one(first);
  (one(rest), ...);
}

int dtype_code(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return DLT_BF16;
    case at::kHalf: return DLT_FP16;
    case at::kFloat: return DLT_FP32;
    default: break;
  }
  raise_py(PyExc_TypeError, std::string("unsupported dtype ") + c10::toString(t.scalar_type()) + "; expected bfloat16, float16 or float32");
}

void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

Tensor empty(at::IntArrayRef size, at::ScalarType st, const Tensor& like) {
  return Tensor(at::detail::empty_cuda(size, st, like.device(), std::nullopt));
}
// torch.empty_like: the strides of a dense tensor are kept
Tensor grad_like(const Tensor& t) { return t.is_contiguous() ? empty(t.sizes(), t.scalar_type(), t) : at::empty_like(t); }

const int64_t* st(const Tensor& t) { return t.strides().data(); }

// ---- which calls the compiled nodes take -----------------------------------------------------------
// Plain eager calls: no trace, transform (torch.func) or dispatch mode is active, the tensors are ordinary strided ones and
// none carries a forward-mode tangent.  Everything else (and its errors) belongs to the autograd.Function classes: a node made
// here would drop the tangent, be missing from the trace, or hide from the mode.
bool plain_keys(c10::DispatchKeySet ks, c10::DispatchKeySet allowed) {
  return (ks.raw_repr() & ~allowed.raw_repr() & ~c10::full_backend_mask) == 0;
}
template <typename... T>
bool plain(const T&... ts) {
  using K = c10::DispatchKey;
  constexpr c10::DispatchKeySet MODES = c10::DispatchKeySet({K::BackendSelect, K::ADInplaceOrView}) | c10::autocast_dispatch_keyset;
  constexpr c10::DispatchKeySet TENSOR = c10::DispatchKeySet({K::Dense, K::ADInplaceOrView, K::AutogradFunctionality}) | c10::autocast_dispatch_keyset;
  auto one = [&](const Tensor& t) { return plain_keys(t.key_set(), TENSOR) && !t._fw_grad(/*level=*/0).defined(); };
  return plain_keys(c10::impl::tls_local_dispatch_key_set().included_, MODES) && (one(ts) && ...);
}

// of those that are there
template <typename... T>
bool plain_each(const T&... ts) { return ((!ts.defined() || plain(ts)) && ...); }

// ---- rotary operands --------------------------------------------------------------------------
struct Rope {
  Tensor idx, row, col;   // row, col: fp32 [len, R, 2] with a contiguous [R, 2] tail
  dlt_rope_t d;
};

Rope make_rope(const Tensor& idx, const Tensor& row, const Tensor& col) {
  require(idx.scalar_type() == at::kInt && idx.dim() == 1 && idx.is_contiguous(), PyExc_TypeError, "idx must be a contiguous 1-D int32 tensor");
  Rope r;
  r.idx = idx;
  auto table = [](const Tensor& t) {
    require(t.dim() == 3 && t.size(2) == 2, PyExc_ValueError, "cos/sin table must have shape [len, R, 2]");
    if (t.scalar_type() == at::kFloat && t.stride(2) == 1 && t.stride(1) == 2) return t;
    return t.to(at::kFloat).contiguous();
  };
  r.row = table(row);
  r.col = table(col);
  r.d.idx = idx.const_data_ptr<int32_t>();
  r.d.row_cs = r.row.const_data_ptr<float>();
  r.d.col_cs = r.col.const_data_ptr<float>();
  r.d.row_cs_stride0 = r.row.stride(0);
  r.d.col_cs_stride0 = r.col.stride(0);
  r.d.n_rdim = (int32_t)r.row.size(1);
  r.d.row_len = (int32_t)r.row.size(0);
  r.d.col_len = (int32_t)r.col.size(0);
  return r;
}

Rope make_rope_for(const Tensor& idx, const Tensor& row, const Tensor& col, const Tensor& like, int64_t n_tokens) {
  if (C10_UNLIKELY(idx.dim() != 1 || idx.size(0) != n_tokens))
    raise_py(PyExc_ValueError, "idx has " + std::to_string(idx.dim() > 0 ? idx.size(0) : 0) + " entries for " + std::to_string(n_tokens) + " tokens");
  require_gpu(like, idx, row, col);
  return make_rope(idx, row, col);
}

// ---- the attention operators --------------------------------------------------------------------
enum class Op { Swa, Image, Flash, Window };

struct Spec {
  Op op = Op::Swa;
  dlt_swa_shape_t swa{};
  dlt_swa_tile_t tile{};
  dlt_flash_shape_t flash{};
  dlt_window_shape_t window{};
  bool narrow = false;   // Swa: see small_tiles
};

Spec swa_spec(const Tensor& q, const Tensor& k, const Tensor& v, const int64_t* dims /* b_size, th, tw, row, col */, double scale) {
  check_assert(q.dim() == 4, "q must have shape [B, H, N, D]");
  const int64_t B = q.size(0), H = q.size(1), N = q.size(2), dk = q.size(3);
  check_assert(N == dims[0] * dims[1] * dims[2], "seqlen should match image size");
  check_assert(k.sizes() == q.sizes() && v.dim() == 4 && v.size(0) == B && v.size(1) == H && v.size(2) == N, "k and v must match q");
  check_assert(q.scalar_type() == k.scalar_type() && k.scalar_type() == v.scalar_type(), "q, k and v must have one dtype");
  Spec s;
  s.op = Op::Swa;
  s.swa = {(int32_t)B, (int32_t)H, (int32_t)dims[0], (int32_t)dims[1], (int32_t)dims[2], (int32_t)dims[3], (int32_t)dims[4],
           (int32_t)dk, (int32_t)v.size(3), (float)scale, dtype_code(q)};
  return s;
}

Spec image_spec(const Tensor& q, const Tensor& k, const Tensor& v, const int64_t* dims /* bh, bw, row, col */, double scale) {
  check_assert(q.dim() == 5, "q must have shape [B, IH, IW, heads, D]");
  const int64_t IH = q.size(1), IW = q.size(2), bh = dims[0], bw = dims[1];
  require(bh != 0 && bw != 0, PyExc_ZeroDivisionError, "tile of zero pixels");
  check_assert(IH % bh == 0 && IW % bw == 0, "image size should be a multiple of the tile size");
  check_assert(k.sizes() == q.sizes() && v.dim() == 5 && v.sizes().slice(0, 4) == q.sizes().slice(0, 4), "k and v must match q");
  check_assert(q.scalar_type() == k.scalar_type() && k.scalar_type() == v.scalar_type(), "q, k and v must have one dtype");
  Spec s;
  s.op = Op::Image;
  s.swa = {(int32_t)q.size(0), (int32_t)q.size(3), (int32_t)(bh * bw), (int32_t)(IH / bh), (int32_t)(IW / bw), (int32_t)dims[2], (int32_t)dims[3],
           (int32_t)q.size(4), (int32_t)v.size(4), (float)scale, dtype_code(q)};
  s.tile = {(int32_t)bh, (int32_t)bw};
  return s;
}

Spec flash_spec(const Tensor& q, const Tensor& k, const Tensor& v, bool causal, double scale) {
  check_assert(q.dim() == 4 && k.dim() == 4 && v.dim() == 4, "q, k and v must have shape [B, H, L, D]");
  check_assert(q.size(3) == k.size(3), "q and k must have one head dim");
  check_assert(q.sizes().slice(0, 2) == k.sizes().slice(0, 2) && q.sizes().slice(0, 2) == v.sizes().slice(0, 2) && k.size(2) == v.size(2),
               "k and v must match q");
  check_assert(q.scalar_type() == k.scalar_type() && k.scalar_type() == v.scalar_type(), "q, k and v must have one dtype");
  Spec s;
  s.op = Op::Flash;
  s.flash = {(int32_t)q.size(0), (int32_t)q.size(1), (int32_t)q.size(2), (int32_t)k.size(2), (int32_t)q.size(3), (int32_t)v.size(3),
             (float)scale, causal ? 1 : 0, dtype_code(q)};
  return s;
}

Spec window_spec(const Tensor& q, const Tensor& k, const Tensor& v, const int64_t* dims /* window, n_sink */, double scale) {
  check_assert(q.dim() == 4 && k.dim() == 4 && v.dim() == 4, "q, k and v must have shape [B, heads, L, D]");
  check_assert(q.size(3) == k.size(3), "q and k must have one head dim");
  check_assert(q.size(0) == k.size(0) && k.sizes().slice(0, 3) == v.sizes().slice(0, 3), "k and v must match q");
  check_assert(q.scalar_type() == k.scalar_type() && k.scalar_type() == v.scalar_type(), "q, k and v must have one dtype");
  for (const Tensor* x : {&q, &k, &v})
    for (int64_t n : x->sizes()) require(n <= INT32_MAX, PyExc_ValueError, "a dim of q, k or v does not fit 32 bits");
  Spec s;
  s.op = Op::Window;
  s.window = {(int32_t)q.size(0), (int32_t)q.size(1), (int32_t)k.size(1), (int32_t)q.size(2), (int32_t)k.size(2), (int32_t)q.size(3), (int32_t)v.size(3),
              (int32_t)dims[0], (int32_t)dims[1], (float)scale, dtype_code(q)};
  return s;
}
// The window and paged kernels read rows in 16-byte pieces, those of 16 tokens and the heads of a group (`G`; keys: 0) at 32-bit offsets.  Anything else is
// copied first, the heads of a token side by side.
bool rows16(const Tensor& x, int64_t G = 0) {
  if (x.dim() != 4 || x.numel() == 0) return true;
  bool ok = (x.stride(3) == 1 || x.size(3) == 1) && (uintptr_t)x.const_data_ptr() % 16 == 0;
  for (int i = 0; i < 3; i++) ok = ok && (x.size(i) == 1 || (x.stride(i) % 8 == 0 && x.stride(i) >= 0));
  auto span = [&](int i, int64_t n) { return x.size(i) == 1 ? 0 : x.stride(i) > ((int64_t)1 << 30) / n ? (int64_t)1 << 30 : n * x.stride(i); };
  return ok && span(2, 17) + (G > 0 ? span(1, G) : 0) < (int64_t)1 << 30;
}
Tensor as_rows16(const Tensor& x, int64_t G = 0) { return rows16(x, G) ? x : x.transpose(1, 2).clone(at::MemoryFormat::Contiguous).transpose(1, 2); }
int64_t group_of(const Tensor& q, const Tensor& k) { return k.dim() == 4 && k.size(1) > 0 ? q.size(1) / k.size(1) : 0; }
// strides of a [.., .., .., D] tensor as the C ABI takes them: those of dims of one element do not matter
std::array<int64_t, 4> st16(const Tensor& x) {
  std::array<int64_t, 4> s;
  for (int i = 0; i < 4; i++) s[i] = i == 3 ? 1 : x.size(i) == 1 || x.numel() == 0 ? 0 : x.stride(i);
  return s;
}

// Partial results of a flash pass that splits its other side: from the caching allocator, on the call's stream, for the call alone.
struct Workspace {
  Tensor t;
  void* ptr = nullptr;
  int64_t bytes = 0;
};
Workspace flash_workspace(const dlt_flash_shape_t& shape, int backward, const Tensor& like) {
  Workspace w;
  check_rc(dlt_flash_workspace(&shape, backward, &w.bytes));
  if (w.bytes > 0) {
    w.t = empty({w.bytes / 4}, at::kFloat, like);
    w.ptr = w.t.mutable_data_ptr();
  }
  return w;
}

Workspace window_workspace(const dlt_window_shape_t& shape, int backward, const Tensor& like) {
  Workspace w;
  check_rc(dlt_window_workspace(&shape, backward, &w.bytes));
  if (w.bytes > 0) {
    w.t = empty({w.bytes / 4}, at::kFloat, like);
    w.ptr = w.t.mutable_data_ptr();
  }
  return w;
}

// The C ABI takes one sequence or more; what else is wrong with a call of none is refused as it would be with one.
void empty_batch(dlt_window_shape_t shape) {
  int64_t bytes;
  shape.B = 1;
  check_rc(dlt_window_workspace(&shape, 0, &bytes));
}

struct Forward { Tensor o, lse, q_rot, k_rot, low; };

// keep_rot: the rotated q and k are stored as well (for the backward pass)
Forward run_forward(const Spec& s, const Tensor& q, const Tensor& k, const Tensor& v, const Rope* rope, bool keep_rot, bool want_lse = true /* Window */) {
  require_gpu(q, k, v);
  c10::DeviceGuard guard(q.device());
  Forward f;
  const at::ScalarType dt = q.scalar_type();
  void* stream = stream_of(q);
  if (s.op == Op::Flash) {
    f.o = empty({q.size(0), q.size(1), q.size(2), v.size(3)}, dt, q);
    f.lse = empty({q.size(0), q.size(1), q.size(2)}, at::kFloat, q);
    const Workspace ws = flash_workspace(s.flash, 0, q);
    check_rc(dlt_flash_fwd_ws(q.const_data_ptr(), st(q), k.const_data_ptr(), st(k), v.const_data_ptr(), st(v), f.o.mutable_data_ptr(), st(f.o),
                              (float*)f.lse.mutable_data_ptr(), st(f.lse), &s.flash, ws.ptr, ws.bytes, stream));
    return f;
  }
  if (s.op == Op::Window && s.window.B == 0) {
    empty_batch(s.window);
    f.o = empty({0, q.size(1), q.size(2), v.size(3)}, dt, q);
    f.lse = empty({0}, at::kFloat, q);
    return f;
  }
  if (s.op == Op::Window) {
    const Workspace ws = window_workspace(s.window, 0, q);
    f.o = empty({q.size(0), q.size(1), q.size(2), v.size(3)}, dt, q);
    if (want_lse) {
      f.lse = empty({q.size(0), k.size(1), q.size(2), q.size(1) / k.size(1)}, at::kFloat, q);
      int32_t tokens = 0;
      check_rc(dlt_window_low_tokens(&s.window, &tokens));
      if (tokens > 0) f.low = empty({q.size(0), q.size(1), tokens, v.size(3)}, dt, q);
    }
    check_rc(dlt_window_fwd(q.const_data_ptr(), st16(q).data(), k.const_data_ptr(), st16(k).data(), v.const_data_ptr(), st16(v).data(), f.o.mutable_data_ptr(),
                            st16(f.o).data(), f.low.defined() ? f.low.mutable_data_ptr() : nullptr, want_lse ? (float*)f.lse.mutable_data_ptr() : nullptr, &s.window, ws.ptr, ws.bytes, stream));
    return f;
  }
  if (s.op == Op::Image) {
    f.o = empty({q.size(0), q.size(1), q.size(2), q.size(3), v.size(4)}, dt, q);
    f.lse = empty({q.size(0), q.size(3), q.size(1) * q.size(2)}, at::kFloat, q);
    check_rc(dlt_swa_fwd_image(q.const_data_ptr(), st(q), k.const_data_ptr(), st(k), v.const_data_ptr(), st(v), f.o.mutable_data_ptr(), st(f.o),
                               (float*)f.lse.mutable_data_ptr(), st(f.lse), &s.swa, &s.tile, nullptr, stream));
    return f;
  }
  f.o = empty({q.size(0), q.size(1), q.size(2), v.size(3)}, dt, q);
  f.lse = empty({q.size(0), q.size(1), q.size(2)}, at::kFloat, q);
  if (keep_rot) {
    f.q_rot = empty(q.sizes(), dt, q);
    f.k_rot = empty(k.sizes(), dt, q);
    check_rc(dlt_swa_fwd_rot(q.const_data_ptr(), st(q), k.const_data_ptr(), st(k), v.const_data_ptr(), st(v), f.o.mutable_data_ptr(), st(f.o),
                             (float*)f.lse.mutable_data_ptr(), st(f.lse), f.q_rot.mutable_data_ptr(), st(f.q_rot), f.k_rot.mutable_data_ptr(),
                             st(f.k_rot), &s.swa, &rope->d, stream));
  } else {
    if (s.narrow)
      check_rc(dlt_swa_fwd_narrow(q.const_data_ptr(), st(q), k.const_data_ptr(), st(k), v.const_data_ptr(), st(v), f.o.mutable_data_ptr(), st(f.o),
                                  (float*)f.lse.mutable_data_ptr(), st(f.lse), &s.swa, stream));
    else
      check_rc(dlt_swa_fwd(q.const_data_ptr(), st(q), k.const_data_ptr(), st(k), v.const_data_ptr(), st(v), f.o.mutable_data_ptr(), st(f.o),
                           (float*)f.lse.mutable_data_ptr(), st(f.lse), &s.swa, rope ? &rope->d : nullptr, stream));
  }
  return f;
}

// rotated: q and k are the rotated tensors that the forward pass kept
std::array<Tensor, 3> run_backward(const Spec& s, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& o, const Tensor& lse,
                                   const Tensor& d_o, const Rope* rope, bool rotated, const Tensor& low = Tensor() /* Window */) {
  require_gpu(q, k, v, o, lse, d_o);
  c10::DeviceGuard guard(q.device());
  void* stream = stream_of(q);
  if (s.op == Op::Window && s.window.B == 0) return {empty(q.sizes(), q.scalar_type(), q), empty(k.sizes(), k.scalar_type(), k), empty(v.sizes(), v.scalar_type(), v)};
  if (s.op == Op::Window) {
    const Workspace ws = window_workspace(s.window, 1, q);
    Tensor dq = empty(q.sizes(), q.scalar_type(), q), dk = empty(k.sizes(), k.scalar_type(), k), dv = empty(v.sizes(), v.scalar_type(), v);
    Tensor delta = empty(lse.sizes(), at::kFloat, lse);
    const Tensor g = as_rows16(d_o, group_of(q, k));
    check_rc(dlt_window_bwd(q.const_data_ptr(), st16(q).data(), k.const_data_ptr(), st16(k).data(), v.const_data_ptr(), st16(v).data(), o.const_data_ptr(),
                            st16(o).data(), low.defined() ? low.const_data_ptr() : nullptr, g.const_data_ptr(), st16(g).data(), (const float*)lse.const_data_ptr(), (float*)delta.mutable_data_ptr(),
                            dq.mutable_data_ptr(), st16(dq).data(), dk.mutable_data_ptr(), st16(dk).data(), dv.mutable_data_ptr(), st16(dv).data(), &s.window,
                            ws.ptr, ws.bytes, stream));
    return {dq, dk, dv};
  }
  Tensor dq = grad_like(q), dk = grad_like(k), dv = grad_like(v), delta = grad_like(lse);
  auto call = [&](auto fn, auto... shape) {
    check_rc(fn(q.const_data_ptr(), st(q), k.const_data_ptr(), st(k), v.const_data_ptr(), st(v), o.const_data_ptr(), st(o), d_o.const_data_ptr(),
                st(d_o), (const float*)lse.const_data_ptr(), (float*)delta.mutable_data_ptr(), st(lse), dq.mutable_data_ptr(), st(dq),
                dk.mutable_data_ptr(), st(dk), dv.mutable_data_ptr(), st(dv), shape..., stream));
  };
  const dlt_rope_t* none = nullptr;
  if (s.op == Op::Flash) {
    const Workspace ws = flash_workspace(s.flash, 1, q);
    call(dlt_flash_bwd_ws, &s.flash, ws.ptr, ws.bytes);
  }
  else if (s.op == Op::Image) call(dlt_swa_bwd_image, &s.swa, &s.tile, none);
  else if (rotated) call(dlt_swa_bwd_rot, &s.swa, (const dlt_rope_t*)&rope->d);
  else if (s.narrow) call(dlt_swa_bwd_narrow, &s.swa);
  else call(dlt_swa_bwd, &s.swa, rope ? (const dlt_rope_t*)&rope->d : none);
  return {dq, dk, dv};
}

// ---- head dims outside the tuned shapes -----------------------------------------------------------
// {dk, dv} to pad q / k and v to before the launch.  Zero columns appended to q, k, v (and to dO) change no score and no
// output column; the copies cost a few percent of what the generic kernels would.
struct Pad { int64_t dk, dv; };

// The token-grid kernels (b_size == 1) take head dims that are multiples of 32 with both in one class (both <= 64, or
// both in 65 ... 128): anything else runs 6 to 9 times slower on the generic kernels.  Tiles of 2 ... 15 tokens run on the
// streaming kernels at head dim 64 or 128 exactly (2 to 4 times).  Tiles of 16 k tokens are padded inside their kernels.
Pad swa_pad(int64_t dk, int64_t dv, at::ScalarType dt, int64_t b_size) {
  const int64_t big = std::max(dk, dv);
  if ((dt != at::kBFloat16 && dt != at::kHalf) || big > 128) return {dk, dv};
  if (2 <= b_size && b_size <= 15) return big <= 64 ? Pad{64, 64} : Pad{128, 128};
  if (b_size != 1) return {dk, dv};
  auto up = [](int64_t d) { return (d + 31) / 32 * 32; };
  return big <= 64 ? Pad{up(dk), up(dv)} : Pad{std::max<int64_t>(96, up(dk)), std::max<int64_t>(96, up(dv))};
}

// Tiles of 2 ... 15 tokens at smaller head dims whose rows can be read in 16-byte pieces as they lie run there without padding (d = 32, 16 heads of 20 x 6
// tiles of 4: the copies around the kernels were 22 of 35 us of host time in the forward pass).
bool rows_of_pieces(const Tensor& x) {
  return x.dim() == 4 && x.size(3) % 8 == 0 && x.stride(3) == 1 && (uintptr_t)x.const_data_ptr() % 16 == 0 && x.stride(0) % 8 == 0 && x.stride(1) % 8 == 0 &&
         x.stride(2) % 8 == 0 && x.stride(2) >= 0 && (x.size(2) + 64) * std::max<int64_t>(x.stride(2), 64) < ((int64_t)1 << 30);
}
bool small_tiles(const Tensor& q, const Tensor& k, const Tensor& v, int64_t b_size, double scale) {
  const at::ScalarType dt = q.scalar_type();
  return 2 <= b_size && b_size <= 15 && (dt == at::kBFloat16 || dt == at::kHalf) && scale > 0 && q.size(-1) <= 64 && v.size(-1) <= 64 &&
         rows_of_pieces(q) && rows_of_pieces(k) && rows_of_pieces(v);
}

// The flash kernels read 16-byte row pieces: head dims that are not multiples of 8 run 3 to 6 times slower on the generic ones.
Pad flash_pad(int64_t dk, int64_t dv, at::ScalarType dt) {
  if ((dt != at::kBFloat16 && dt != at::kHalf) || std::max(dk, dv) > 128) return {dk, dv};
  return {(dk + 7) / 8 * 8, (dv + 7) / 8 * 8};
}

Tensor pad_last(const Tensor& x, int64_t d) { return x.size(-1) == d ? x : at::constant_pad_nd(x, {0, d - x.size(-1)}); }
Tensor cut_last(const Tensor& x, int64_t d) { return x.size(-1) == d ? x : x.narrow(-1, 0, d).contiguous(); }

// ---- autograd ---------------------------------------------------------------------------------------
// A leaf keeps one accumulation node while any graph of it lives, with the stream that was current when the node was made.  A backward pass that is being captured
// cannot pass a gradient to one of the default stream: the engine would make the two streams wait for each other, which ends the capture, and on ROCm the process.
void check_capture(Node& node) {
  bool on_default = false;
  for (size_t i = 0; i < node.num_outputs(); i++) {
    if (!node.task_should_compute_output(i)) continue;   // this pass asks for no gradient behind that input: the engine passes none on
    const std::optional<c10::Stream> s = node.next_edge(i).function->stream();
    on_default = on_default || (s.has_value() && s->id() == 0);
  }
  if (C10_UNLIKELY(on_default && c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None))
    raise_py(PyExc_RuntimeError, "a captured backward pass reaches a leaf that belongs to a graph of the default stream: release that graph (the tensors made from the "
                                 "leaf outside the capture), or make it on another stream");
}
// first derivatives only: a second one raises where it is asked for (without a graph it would be dropped in silence)
void differentiable_once(variable_list& grads) {
  if (C10_LIKELY(!at::GradMode::is_enabled())) return;
  std::shared_ptr<torch::autograd::DelayedError> once(
      new torch::autograd::DelayedError("trying to differentiate twice a function that was marked with @once_differentiable", (int64_t)grads.size()), torch::autograd::deleteNode);
  for (Tensor& g : grads) g = g.detach().requires_grad_(true);
  grads = (*once)(std::move(grads));
}

struct AttnBackward : public Node {
  Spec spec;
  bool has_rope = false, rotated = false;
  int64_t dk = 0, dv = 0;   // head dims of the caller's tensors
  SavedVariable q, k, v, o, lse, idx, row, col, low;

  std::string name() const override { return "DltAttentionBackward"; }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    for (SavedVariable* s : {&q, &k, &v, &o, &lse, &idx, &row, &col, &low}) s->reset_data();
  }
  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    if (spec.op == Op::Window) check_capture(*this);
    if (!grads[0].defined()) grads[0] = input_metadata(0).zeros_like();   // as torch.autograd.Function does
    // Unpacked with autograd as it is: an unpack hook may run the forward pass again (activation checkpointing), and what it runs
    // has to be recorded.
    Tensor q_ = q.unpack(), k_ = k.unpack(), v_ = v.unpack(), o_ = o.unpack(shared_from_this()), lse_ = lse.unpack();
    Tensor idx_, row_, col_, low_;
    if (spec.op == Op::Window) low_ = low.unpack();
    if (has_rope) {
      idx_ = idx.unpack();
      row_ = row.unpack();
      col_ = col.unpack();
    }
    variable_list out;
    {
      at::AutoDispatchBelowADInplaceOrView below;
      Rope rope;
      if (has_rope) rope = make_rope_for(idx_, row_, col_, q_, q_.size(2));
      Tensor d_o = pad_last(grads[0], v_.size(-1));
      if (spec.narrow && !rows_of_pieces(d_o)) d_o = d_o.contiguous();
      if (spec.op == Op::Window) {   // what an unpack hook gives need not lie as what was packed
        q_ = as_rows16(q_, group_of(q_, k_));
        k_ = as_rows16(k_);
        v_ = as_rows16(v_);
        o_ = as_rows16(o_);
        lse_ = lse_.contiguous();
        if (low_.defined()) low_ = low_.contiguous();
      }
      auto g = run_backward(spec, q_, k_, v_, o_, lse_, d_o, has_rope ? &rope : nullptr, rotated, low_);
      out = {cut_last(g[0], dk), cut_last(g[1], dk), cut_last(g[2], dv)};
    }
    if (spec.op == Op::Window) differentiable_once(out);
    return out;
  }
};

struct RopeBackward : public Node {
  SavedVariable idx, row, col;
  std::string name() const override { return "DltRotaryPE2DBackward"; }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    idx.reset_data();
    row.reset_data();
    col.reset_data();
  }
  variable_list apply(variable_list&& grads) override;
};

template <typename N>
std::shared_ptr<N> make_node() { return std::shared_ptr<N>(new N(), torch::autograd::deleteNode); }

// Forward pass with the graph recorded when q, k or v asks for it (graph == false: never).
Tensor attention(Op op, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor* rope_t, const int64_t* dims, bool causal, double scale,
                 bool keep_rot, bool graph) {
  std::shared_ptr<AttnBackward> node;
  const bool grad = graph && torch::autograd::compute_requires_grad(q, k, v);
  if (grad) {
    node = make_node<AttnBackward>();
    node->set_next_edges(torch::autograd::collect_next_edges(q, k, v));
  }
  pybind11::gil_scoped_release nogil;
  Tensor out, pq = q, pk = k, pv = v;
  Forward f;
  Spec spec;
  check_assert(q.dim() >= 2 && k.dim() == q.dim() && v.dim() == q.dim(), "q, k and v must have the same number of dims");
  const int64_t dk = q.size(-1), dv = v.size(-1);
  {
    at::AutoDispatchBelowADInplaceOrView below;
    const bool narrow = op == Op::Swa && rope_t == nullptr && small_tiles(q, k, v, dims[0], scale);
    const Pad pad = narrow ? Pad{dk, dv} : op == Op::Flash || op == Op::Window ? flash_pad(dk, dv, q.scalar_type()) : op == Op::Swa ? swa_pad(dk, dv, q.scalar_type(), dims[0]) : Pad{dk, dv};
    if (C10_UNLIKELY(pad.dk != dk || pad.dv != dv)) {
      pq = pad_last(q, pad.dk);
      pk = pad_last(k, pad.dk);
      pv = pad_last(v, pad.dv);
    }
    if (op == Op::Window) {
      check_assert(q.dim() == 4, "q, k and v must have shape [B, heads, L, D]");
      require_gpu(q, k, v);
      pq = as_rows16(pq, group_of(pq, pk));
      pk = as_rows16(pk);
      pv = as_rows16(pv);
    }
    spec = op == Op::Window ? window_spec(pq, pk, pv, dims, scale) : op == Op::Flash ? flash_spec(pq, pk, pv, causal, scale) : op == Op::Image ? image_spec(pq, pk, pv, dims, scale) : swa_spec(pq, pk, pv, dims, scale);
    spec.narrow = narrow;
    Rope rope;
    if (rope_t != nullptr) {
      check_assert(rope_t[1].dim() == 3 && rope_t[2].dim() == 3 && rope_t[1].size(1) == rope_t[2].size(1), "row and column table must have one R");
      check_assert(rope_t[0].dim() == 1 && rope_t[0].size(0) == pq.size(2), "idx must have one entry per token");
      require_gpu(pq, pk, pv);
      rope = make_rope_for(rope_t[0], rope_t[1], rope_t[2], pq, pq.size(2));
    }
    f = run_forward(spec, pq, pk, pv, rope_t ? &rope : nullptr, keep_rot, grad);
    out = cut_last(f.o, dv);
  }
  // saved with autograd as it is: pack hooks are the caller's code
  if (grad) {
    node->spec = spec;
    node->dk = dk;
    node->dv = dv;
    node->q = SavedVariable(keep_rot ? f.q_rot : pq, false);
    node->k = SavedVariable(keep_rot ? f.k_rot : pk, false);
    node->v = SavedVariable(pv, false);
    node->lse = SavedVariable(f.lse, false);
    node->low = SavedVariable(f.low, false);
    if (rope_t != nullptr) {
      node->has_rope = true;
      node->rotated = keep_rot;
      node->idx = SavedVariable(rope_t[0], false);
      node->row = SavedVariable(rope_t[1], false);
      node->col = SavedVariable(rope_t[2], false);
    }
    const bool whole = out.is_same(f.o);
    if (!whole) node->o = SavedVariable(f.o, false);
    torch::autograd::set_history(out, node);
    if (whole) node->o = SavedVariable(out, true);
  }
  return out;
}

// ---- rotation -----------------------------------------------------------------------------------------
// {batch stride, token stride, element stride} and batch rows of x[..., N, C] when the leading dims are one run
struct Rows { int64_t s[3], nb; };
bool rows_of(const Tensor& x, Rows& r) {
  const int64_t nd = x.dim();
  r.nb = 1;
  r.s[0] = 0;
  for (int64_t i = nd - 3; i >= 0; i--) {
    if (x.size(i) == 1) continue;
    if (r.nb == 1) r.s[0] = x.stride(i);
    else if (x.stride(i) != r.nb * r.s[0]) return false;
    r.nb *= x.size(i);
  }
  r.s[1] = x.stride(nd - 2);
  r.s[2] = x.stride(nd - 1);
  return true;
}

void rotate_inplace(const Tensor& x, const Rows& r, const Rope& rope, bool inverse) {
  c10::DeviceGuard guard(x.device());
  check_rc(dlt_rope2d(x.mutable_data_ptr(), r.s, r.nb, x.size(-2), x.size(-1), &rope.d, inverse, dtype_code(x), stream_of(x)));
}

variable_list RopeBackward::apply(variable_list&& grads) {
  std::lock_guard<std::mutex> lock(mutex_);
  if (!grads[0].defined()) grads[0] = input_metadata(0).zeros_like();
  const Tensor idx_ = idx.unpack(), row_ = row.unpack(), col_ = col.unpack();   // before the guard: see AttnBackward
  Tensor dy = grads[0], dx;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    const Rope rope = make_rope(idx_, row_, col_);
    require_gpu(dy, rope.idx, rope.row, rope.col);
    Rows rs, rd;
    if (!rows_of(dy, rs)) {
      dy = dy.contiguous();
      rows_of(dy, rs);
    }
    c10::DeviceGuard guard(dy.device());
    dx = empty(dy.sizes(), dy.scalar_type(), dy);
    rows_of(dx, rd);
    check_rc(dlt_rope2d_copy(dy.const_data_ptr(), rs.s, dx.mutable_data_ptr(), rd.s, rd.nb, dy.size(-2), dy.size(-1), &rope.d, 1, dtype_code(dy),
                             stream_of(dy)));
  }
  // differentiable once: a second derivative raises where it is asked for (without a graph it would be dropped in silence)
  if (C10_UNLIKELY(at::GradMode::is_enabled() && grads[0].requires_grad())) {
    std::shared_ptr<torch::autograd::DelayedError> once(
        new torch::autograd::DelayedError("trying to differentiate twice a function that was marked with @once_differentiable", 1), torch::autograd::deleteNode);
    return (*once)({dx.detach().requires_grad_(true)});
  }
  return {dx};
}

// x[..., N, C] is rotated in place; the graph sees an in-place operation on x
void rope_apply(const Tensor& x, const Rows& r, const Tensor& idx, const Tensor& row, const Tensor& col) {
  check_assert(row.dim() == 3 && col.dim() == 3 && row.size(1) == col.size(1), "row and column table must have one R");
  check_assert(idx.dim() == 1 && idx.size(0) == x.size(-2), "idx must have one entry per token");
  require_gpu(x, idx, row, col);
  const bool grad = torch::autograd::compute_requires_grad(x);
  torch::autograd::check_inplace(x, grad);
  std::shared_ptr<RopeBackward> node;
  if (grad) {
    node = make_node<RopeBackward>();
    node->set_next_edges(torch::autograd::collect_next_edges(x));
    node->idx = SavedVariable(idx, false);
    node->row = SavedVariable(row, false);
    node->col = SavedVariable(col, false);
  }
  {
    at::AutoDispatchBelowADInplaceOrView below;
    rotate_inplace(x, r, make_rope(idx, row, col), false);
  }
  torch::autograd::increment_version(x);
  if (grad) torch::autograd::rebase_history(x, node);
}

// ---- rotation with several axes -------------------------------------------------------------------------
// tensors that a call writes: no element twice
void check_written(const Tensor& x, const char* name) {
  if (C10_UNLIKELY(at::has_internal_overlap(x) == at::MemOverlap::Yes)) raise_py(PyExc_RuntimeError, std::string(name) + " has elements that share memory (an expanded tensor): it cannot be written in place");
}
// Is some element of x one of y?  With x[i] at sum i_d s_d and y[j] at D + sum j_d s'_d that asks for whole numbers with sum i_d s_d - sum j_d s'_d = D.  Strides from the
// largest on; a number is tried only where the strides behind it can make up the rest, which leaves one or two for dims that lie inside each other.  Layouts that need
// more than a few thousand tries are taken as apart.
struct Meeting {
  struct Dim { int64_t stride, lo, hi; };   // the sum of the dims of both tensors with this stride
  Dim d[8];
  int n = 0, tries = 4096;
  void add(const Tensor& x, bool second) {
    for (int64_t i = 0; i < x.dim() && i < 4; i++) {
      const int64_t s = x.stride(i), m = x.size(i) - 1;
      if (s == 0 || m == 0) continue;
      int k = 0;
      while (k < n && d[k].stride != s) k++;
      if (k == n) d[n++] = {s, 0, 0};
      (second ? d[k].lo : d[k].hi) += second ? -m : m;
    }
  }
  bool solve(int k, int64_t rest) {
    if (k == n) return rest == 0;
    if (--tries < 0) return false;
    int64_t lo = 0, hi = 0;   // what the dims behind this one can add
    for (int i = k + 1; i < n; i++) { lo += d[i].stride * d[i].lo; hi += d[i].stride * d[i].hi; }
    auto floor_div = [](int64_t a, int64_t b) { return a / b - (a % b < 0); };
    const int64_t t0 = std::max(d[k].lo, -floor_div(hi - rest, d[k].stride)), t1 = std::min(d[k].hi, floor_div(rest - lo, d[k].stride));
    for (int64_t t = t0; t <= t1 && tries >= 0; t++)
      if (solve(k + 1, rest - t * d[k].stride)) return true;
    return false;
  }
};
bool meet(const Tensor& x, const Tensor& y) {
  if (x.numel() == 0 || y.numel() == 0) return false;
  auto bytes = [](const Tensor& t) {
    int64_t n = 1;
    for (int64_t i = 0; i < t.dim(); i++) n += (t.size(i) - 1) * t.stride(i);
    return n * (int64_t)t.element_size();
  };
  const char *px = (const char*)x.const_data_ptr(), *py = (const char*)y.const_data_ptr();
  if (px + bytes(x) <= py || py + bytes(y) <= px) return false;
  const int64_t es = (int64_t)x.element_size();   // one dtype
  if ((py - px) % es != 0) return true;
  Meeting m;
  m.add(x, false);
  m.add(y, true);
  std::sort(m.d, m.d + m.n, [](const Meeting::Dim& a, const Meeting::Dim& b) { return a.stride > b.stride; });
  return m.solve(0, (py - px) / es);
}
void check_two(const Tensor& x, const Tensor& y, const char* names) {
  if (C10_UNLIKELY(x.numel() > 0 && y.numel() > 0 && x.const_data_ptr() == y.const_data_ptr())) raise_py(PyExc_RuntimeError, std::string(names) + " must be two tensors");
  if (C10_UNLIKELY(meet(x, y))) raise_py(PyExc_RuntimeError, std::string(names) + " share memory: they cannot be written in one call");
}

struct Axes {
  Tensor pos;                   // int32 [axes, N] or [axes, B, N]
  std::vector<Tensor> tables;   // fp32 [len, R, 2]
  int layout = DLT_ROPE_BLOCKS;
};

// n_tokens, batch: those of the tensors; `d` holds pointers into `t`, whose tables it may replace by dense fp32 copies
void make_axes(Axes& t, int64_t batch, int64_t n_tokens, const Tensor& like, dlt_rope_axes_t& d) {
  d = {};
  require(!t.tables.empty() && t.tables.size() <= DLT_ROPE_AXES_MAX, PyExc_ValueError, "one to four axes are supported");
  d.n_axes = (int32_t)t.tables.size();
  d.layout = t.layout;
  if (t.pos.defined()) {
    require(t.pos.scalar_type() == at::kInt && (t.pos.dim() == 2 || t.pos.dim() == 3), PyExc_TypeError, "pos must be an int32 tensor [axes, N] or [axes, B, N]");
    require(t.pos.size(0) == d.n_axes && t.pos.size(-1) == n_tokens && (t.pos.dim() == 2 || t.pos.size(1) == batch), PyExc_ValueError,
            "pos must have an entry for every axis and token");
    require_gpu(like, t.pos);
    d.pos = t.pos.const_data_ptr<int32_t>();
    d.pos_strides[0] = t.pos.stride(0);
    d.pos_strides[1] = t.pos.dim() == 3 ? t.pos.stride(1) : 0;
    d.pos_strides[2] = t.pos.stride(-1);
  }
  for (int i = 0; i < d.n_axes; i++) {
    Tensor& x = t.tables[i];
    require(x.dim() == 3 && x.size(2) == 2, PyExc_ValueError, "cos/sin table must have shape [len, R, 2]");
    require_gpu(like, x);
    const bool dense = x.scalar_type() == at::kFloat && (x.numel() == 0 || (x.stride(2) == 1 && (x.size(1) == 1 || x.stride(1) == 2) && x.stride(0) % 2 == 0 &&
                                                         x.stride(0) >= 2 * x.size(1) && (uintptr_t)x.const_data_ptr() % 8 == 0));
    if (!dense) x = x.to(at::kFloat).clone(at::MemoryFormat::Contiguous);
    d.table[i] = (const float*)x.const_data_ptr();
    d.table_stride0[i] = std::max<int64_t>(x.size(0) == 1 ? 2 * x.size(1) : x.stride(0), 2 * x.size(1));
    d.n_rdim[i] = (int32_t)x.size(1);
    d.len[i] = (int32_t)x.size(0);
  }
}

// q and k (k undefined: q alone) into q_out and k_out, which may be q and k themselves
void run_axes(const Tensor& q, const Tensor& k, const Tensor& q_out, const Tensor& k_out, Axes t, bool inverse) {
  check_assert(q.dim() == 4 && (!k.defined() || k.dim() == 4), "q and k must have shape [B, heads, N, C]");
  check_assert(!k.defined() || (k.size(0) == q.size(0) && k.size(2) == q.size(2) && k.size(3) == q.size(3) && k.scalar_type() == q.scalar_type()),
               "q and k must have one batch, token count, head dim and dtype");
  check_assert(t.pos.defined(), "pos is needed");
  for (const Tensor* x : {&q, &k})
    if (x->defined())
      for (int64_t n : x->sizes()) require(n <= INT32_MAX, PyExc_ValueError, "a dim of q or k does not fit 32 bits");
  if (k.defined()) require_gpu(q, k);
  else require_gpu(q);
  dlt_rope_axes_t d;
  make_axes(t, q.size(0), q.size(2), q, d);
  c10::DeviceGuard guard(q.device());
  check_rc(dlt_rope_axes(q.const_data_ptr(), st(q), q_out.mutable_data_ptr(), st(q_out), (int32_t)q.size(1), k.defined() ? k.const_data_ptr() : nullptr,
                         k.defined() ? st(k) : nullptr, k.defined() ? k_out.mutable_data_ptr() : nullptr, k.defined() ? st(k_out) : nullptr,
                         k.defined() ? (int32_t)k.size(1) : 0, (int32_t)q.size(0), q.size(2), q.size(3), &d, inverse, dtype_code(q), stream_of(q)));
}
std::array<Tensor, 2> run_axes_new(const Tensor& q, const Tensor& k, const Axes& t, bool inverse) {
  if (k.defined()) require_gpu(q, k);
  else require_gpu(q);
  c10::DeviceGuard guard(q.device());
  std::array<Tensor, 2> out{empty(q.sizes(), q.scalar_type(), q), k.defined() ? empty(k.sizes(), k.scalar_type(), k) : Tensor()};
  run_axes(q, k, out[0], out[1], t, inverse);
  return out;
}

std::array<Tensor, 2> rope_axes(const Tensor& q, const Tensor& k, const Axes& t, bool inverse);

struct RopeAxesBackward : public Node {
  SavedVariable pos;
  std::vector<SavedVariable> tables;
  int layout = 0;
  bool inverse = false, pair = false;
  std::string name() const override { return "DltRopeAxesBackward"; }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    pos.reset_data();
    for (SavedVariable& s : tables) s.reset_data();
  }
  // The backward pass of a rotation is the inverse one: the same operator, which records its own graph where one is wanted.
  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    check_capture(*this);
    Axes t;
    t.pos = pos.unpack();
    for (SavedVariable& s : tables) t.tables.push_back(s.unpack());
    t.layout = layout;
    const bool a = grads[0].defined(), b = pair && grads[1].defined();
    variable_list out(pair ? 2 : 1);
    if (a && b) {
      auto g = rope_axes(grads[0], grads[1], t, !inverse);
      out[0] = g[0];
      out[1] = g[1];
    } else if (a || b) {
      out[a ? 0 : 1] = rope_axes(grads[a ? 0 : 1], Tensor(), t, !inverse)[0];
    }
    return out;
  }
};

// rotated copies, with the graph recorded when q or k asks for it
std::array<Tensor, 2> rope_axes(const Tensor& q, const Tensor& k, const Axes& t, bool inverse) {
  const bool pair = k.defined();
  std::shared_ptr<RopeAxesBackward> node;
  if (pair ? torch::autograd::compute_requires_grad(q, k) : torch::autograd::compute_requires_grad(q)) {
    node = make_node<RopeAxesBackward>();
    node->set_next_edges(pair ? torch::autograd::collect_next_edges(q, k) : torch::autograd::collect_next_edges(q));
    node->inverse = inverse;
    node->pair = pair;
    node->layout = t.layout;
  }
  std::array<Tensor, 2> out;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    out = run_axes_new(q, k, t, inverse);
  }
  if (node) {
    node->pos = SavedVariable(t.pos, false);
    for (const Tensor& x : t.tables) node->tables.emplace_back(x, false);
    torch::autograd::set_history(out[0], node);
    if (pair) torch::autograd::set_history(out[1], node);
  }
  return out;
}

// ---- the paged cache ---------------------------------------------------------------------------------------
struct Paged {
  dlt_paged_shape_t s{};
  const int32_t *table = nullptr, *seq = nullptr, *n_new = nullptr;
  int64_t ts = 0;
};
// dtype: of the new tokens (-1: the cache's)
Paged paged_args(const Tensor& kc, const Tensor& vc, const Tensor& table, const Tensor& seq, const Tensor* n_new, int64_t B, int64_t T, int64_t H, int dtype = -1) {
  check_assert(kc.dim() == 4 && vc.dim() == 4 && kc.sizes().slice(0, 3) == vc.sizes().slice(0, 3), "caches must have shape [pages, heads, page, D], all but D alike");
  check_assert(kc.scalar_type() == vc.scalar_type(), "caches must have one dtype");
  require(table.scalar_type() == at::kInt && table.dim() == 2 && (table.size(1) <= 1 || table.stride(1) == 1), PyExc_TypeError,
          "page_table must be an int32 tensor [B, pages of a sequence] with contiguous rows");
  require(seq.scalar_type() == at::kInt && seq.dim() == 1 && (seq.size(0) <= 1 || seq.stride(0) == 1), PyExc_TypeError, "seq_len must be a contiguous 1-D int32 tensor");
  check_assert(table.size(0) == B && seq.size(0) == B, "page_table and seq_len must have a row for every sequence");
  require_gpu(kc, vc, table, seq);
  Paged p;
  if (n_new != nullptr) {
    require(n_new->scalar_type() == at::kInt && n_new->dim() == 1 && (n_new->size(0) <= 1 || n_new->stride(0) == 1), PyExc_TypeError,
            "n_new must be a contiguous 1-D int32 tensor");
    check_assert(n_new->size(0) == B, "n_new must have an entry for every sequence");
    require_gpu(kc, *n_new);
    p.n_new = n_new->const_data_ptr<int32_t>();
  }
  check_assert(kc.size(0) <= INT32_MAX && kc.size(2) <= INT32_MAX && table.size(1) <= INT32_MAX && T <= INT32_MAX, "too many pages or tokens");
  p.table = table.const_data_ptr<int32_t>();
  p.seq = seq.const_data_ptr<int32_t>();
  p.ts = table.stride(0);
  p.s.B = (int32_t)B; p.s.H = (int32_t)H; p.s.Hkv = (int32_t)kc.size(1); p.s.T = (int32_t)T;
  p.s.dk = (int32_t)kc.size(3); p.s.dv = (int32_t)vc.size(3);
  p.s.page = (int32_t)kc.size(2); p.s.n_pages = (int32_t)kc.size(0); p.s.cols = (int32_t)table.size(1);
  p.s.dtype = dtype < 0 ? dtype_code(kc) : dtype;
  return p;
}

// ---- arguments --------------------------------------------------------------------------------------------
const Tensor& tensor_arg(PyObject* o) {
  if (C10_UNLIKELY(!THPVariable_Check(o))) raise_py(PyExc_TypeError, std::string("expected a tensor, got ") + Py_TYPE(o)->tp_name);
  return THPVariable_Unpack(o);
}

int64_t int_arg(PyObject* o) {
  const int64_t v = PyLong_Check(o) ? PyLong_AsLongLong(o) : [&] {
    PyObject* i = PyNumber_Index(o);
    if (i == nullptr) throw python_error();
    const int64_t r = PyLong_AsLongLong(i);
    Py_DECREF(i);
    return r;
  }();
  if (C10_UNLIKELY(v == -1 && PyErr_Occurred())) throw python_error();
  if (C10_UNLIKELY(v < INT32_MIN || v > INT32_MAX)) raise_py(PyExc_OverflowError, "argument does not fit 32 bits");
  return v;
}

double float_arg(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (C10_UNLIKELY(v == -1.0 && PyErr_Occurred())) throw python_error();
  return v;
}

bool bool_arg(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (C10_UNLIKELY(v < 0)) throw python_error();
  return v != 0;
}

void count(Py_ssize_t n, Py_ssize_t lo, Py_ssize_t hi) {
  if (C10_UNLIKELY(n < lo || n > hi)) raise_py(PyExc_TypeError, "takes " + std::to_string(hi) + " positional arguments, got " + std::to_string(n));
}

// ---- entry points: see the Python modules for what they do ----------------------------------------------------
PyObject* py_tiled_swa(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 9, 9);
  int64_t dims[5];
  for (int i = 0; i < 5; i++) dims[i] = int_arg(a[3 + i]);
  if (!plain(tensor_arg(a[0]), tensor_arg(a[1]), tensor_arg(a[2]))) Py_RETURN_NOTIMPLEMENTED;
  return THPVariable_Wrap(attention(Op::Swa, tensor_arg(a[0]), tensor_arg(a[1]), tensor_arg(a[2]), nullptr, dims, false, float_arg(a[8]), false, true));
  END_HANDLE_TH_ERRORS
}

PyObject* py_tiled_swa_fwd(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 9, 9);
  int64_t dims[5];
  for (int i = 0; i < 5; i++) dims[i] = int_arg(a[3 + i]);
  return THPVariable_Wrap(attention(Op::Swa, tensor_arg(a[0]), tensor_arg(a[1]), tensor_arg(a[2]), nullptr, dims, false, float_arg(a[8]), false, false));
  END_HANDLE_TH_ERRORS
}

PyObject* py_tiled_swa_rope(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 12, 13);
  int64_t dims[5];
  for (int i = 0; i < 5; i++) dims[i] = int_arg(a[6 + i]);
  const Tensor rope[3] = {tensor_arg(a[3]), tensor_arg(a[4]), tensor_arg(a[5])};
  if (!plain(tensor_arg(a[0]), tensor_arg(a[1]), tensor_arg(a[2]), rope[0], rope[1], rope[2])) Py_RETURN_NOTIMPLEMENTED;
  const bool keep = n < 13 || a[12] == Py_None || bool_arg(a[12]);
  return THPVariable_Wrap(attention(Op::Swa, tensor_arg(a[0]), tensor_arg(a[1]), tensor_arg(a[2]), rope, dims, false, float_arg(a[11]), keep, true));
  END_HANDLE_TH_ERRORS
}

PyObject* py_tiled_swa_image(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 8, 8);
  int64_t dims[4];
  for (int i = 0; i < 4; i++) dims[i] = int_arg(a[3 + i]);
  if (!plain(tensor_arg(a[0]), tensor_arg(a[1]), tensor_arg(a[2]))) Py_RETURN_NOTIMPLEMENTED;
  return THPVariable_Wrap(attention(Op::Image, tensor_arg(a[0]), tensor_arg(a[1]), tensor_arg(a[2]), nullptr, dims, false, float_arg(a[7]), false, true));
  END_HANDLE_TH_ERRORS
}

PyObject* py_flash(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 5, 5);
  if (!plain(tensor_arg(a[0]), tensor_arg(a[1]), tensor_arg(a[2]))) Py_RETURN_NOTIMPLEMENTED;
  return THPVariable_Wrap(attention(Op::Flash, tensor_arg(a[0]), tensor_arg(a[1]), tensor_arg(a[2]), nullptr, nullptr, bool_arg(a[3]), float_arg(a[4]),
                                    false, true));
  END_HANDLE_TH_ERRORS
}

// (q, k, v, rope or None, keep_rot, B, H, b_size, th, tw, row, col, dk, dv, scale, dtype) -> (o, lse2[, q_rot, k_rot])
// and (q, k, v, o, lse2, do, rope or None, rotated, <the same 11 numbers>) -> (dq, dk, dv): one direction without a graph
Spec swa_spec_from(PyObject* const* a) {
  Spec s;
  s.op = Op::Swa;
  s.swa = {(int32_t)int_arg(a[0]), (int32_t)int_arg(a[1]), (int32_t)int_arg(a[2]), (int32_t)int_arg(a[3]), (int32_t)int_arg(a[4]), (int32_t)int_arg(a[5]),
           (int32_t)int_arg(a[6]), (int32_t)int_arg(a[7]), (int32_t)int_arg(a[8]), (float)float_arg(a[9]), (int32_t)int_arg(a[10])};
  return s;
}

bool rope_arg(PyObject* o, const Tensor& like, Rope& r) {
  if (o == Py_None) return false;
  require(PyTuple_Check(o) && PyTuple_GET_SIZE(o) == 3, PyExc_TypeError, "rope must be (idx, row table, column table)");
  r = make_rope_for(tensor_arg(PyTuple_GET_ITEM(o, 0)), tensor_arg(PyTuple_GET_ITEM(o, 1)), tensor_arg(PyTuple_GET_ITEM(o, 2)), like, like.size(2));
  return true;
}

PyObject* py_swa_forward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 16, 16);
  at::AutoDispatchBelowADInplaceOrView below;
  const Tensor &q = tensor_arg(a[0]), &k = tensor_arg(a[1]), &v = tensor_arg(a[2]);
  require_gpu(q, k, v);
  Rope r;
  const bool rope = rope_arg(a[3], q, r), keep = bool_arg(a[4]);
  const Forward f = run_forward(swa_spec_from(a + 5), q, k, v, rope ? &r : nullptr, keep);
  if (keep) return Py_BuildValue("(NNNN)", THPVariable_Wrap(f.o), THPVariable_Wrap(f.lse), THPVariable_Wrap(f.q_rot), THPVariable_Wrap(f.k_rot));
  return Py_BuildValue("(NN)", THPVariable_Wrap(f.o), THPVariable_Wrap(f.lse));
  END_HANDLE_TH_ERRORS
}

PyObject* py_swa_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 19, 19);
  at::AutoDispatchBelowADInplaceOrView below;
  const Tensor &q = tensor_arg(a[0]), &k = tensor_arg(a[1]), &v = tensor_arg(a[2]), &o = tensor_arg(a[3]), &lse = tensor_arg(a[4]), &d_o = tensor_arg(a[5]);
  Rope r;
  const bool rope = rope_arg(a[6], v, r), rotated = bool_arg(a[7]);
  auto g = run_backward(swa_spec_from(a + 8), q, k, v, o, lse, d_o, rope ? &r : nullptr, rotated);
  return Py_BuildValue("(NNN)", THPVariable_Wrap(g[0]), THPVariable_Wrap(g[1]), THPVariable_Wrap(g[2]));
  END_HANDLE_TH_ERRORS
}

// (q, k, v, bh, bw, row, col, scale) -> (o, lse2) and (q, k, v, o, lse2, do, the same 5 numbers) -> (dq, dk, dv): no graph
PyObject* py_image_forward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 8, 8);
  at::AutoDispatchBelowADInplaceOrView below;
  const Tensor &q = tensor_arg(a[0]), &k = tensor_arg(a[1]), &v = tensor_arg(a[2]);
  const int64_t dims[4] = {int_arg(a[3]), int_arg(a[4]), int_arg(a[5]), int_arg(a[6])};
  const Forward f = run_forward(image_spec(q, k, v, dims, float_arg(a[7])), q, k, v, nullptr, false);
  return Py_BuildValue("(NN)", THPVariable_Wrap(f.o), THPVariable_Wrap(f.lse));
  END_HANDLE_TH_ERRORS
}

PyObject* py_image_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 11, 11);
  at::AutoDispatchBelowADInplaceOrView below;
  const Tensor &q = tensor_arg(a[0]), &k = tensor_arg(a[1]), &v = tensor_arg(a[2]), &o = tensor_arg(a[3]), &lse = tensor_arg(a[4]), &d_o = tensor_arg(a[5]);
  const int64_t dims[4] = {int_arg(a[6]), int_arg(a[7]), int_arg(a[8]), int_arg(a[9])};
  auto g = run_backward(image_spec(q, k, v, dims, float_arg(a[10])), q, k, v, o, lse, d_o, nullptr, false);
  return Py_BuildValue("(NNN)", THPVariable_Wrap(g[0]), THPVariable_Wrap(g[1]), THPVariable_Wrap(g[2]));
  END_HANDLE_TH_ERRORS
}

// (q, k, v, o, M, do, causal, scale) -> (dq, dk, dv) without a graph and without padding
PyObject* py_flash_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 8, 8);
  at::AutoDispatchBelowADInplaceOrView below;
  const Tensor &q = tensor_arg(a[0]), &k = tensor_arg(a[1]), &v = tensor_arg(a[2]), &o = tensor_arg(a[3]), &lse = tensor_arg(a[4]), &d_o = tensor_arg(a[5]);
  auto g = run_backward(flash_spec(q, k, v, bool_arg(a[6]), float_arg(a[7])), q, k, v, o, lse, d_o, nullptr, false);
  return Py_BuildValue("(NNN)", THPVariable_Wrap(g[0]), THPVariable_Wrap(g[1]), THPVariable_Wrap(g[2]));
  END_HANDLE_TH_ERRORS
}

// (q, k, v, causal, scale) -> (o, M) without a graph and without padding
PyObject* py_flash_forward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 5, 5);
  at::AutoDispatchBelowADInplaceOrView below;
  const Tensor &q = tensor_arg(a[0]), &k = tensor_arg(a[1]), &v = tensor_arg(a[2]);
  const Forward f = run_forward(flash_spec(q, k, v, bool_arg(a[3]), float_arg(a[4])), q, k, v, nullptr, false);
  return Py_BuildValue("(NN)", THPVariable_Wrap(f.o), THPVariable_Wrap(f.lse));
  END_HANDLE_TH_ERRORS
}

int32_t window_arg(PyObject* o) { return o == Py_None ? INT32_MAX : (int32_t)int_arg(o); }

// (q, k, v, window or None, n_sink, scale)
PyObject* py_window(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 6, 6);
  const int64_t dims[2] = {window_arg(a[3]), int_arg(a[4])};
  if (!plain(tensor_arg(a[0]), tensor_arg(a[1]), tensor_arg(a[2]))) Py_RETURN_NOTIMPLEMENTED;
  return THPVariable_Wrap(attention(Op::Window, tensor_arg(a[0]), tensor_arg(a[1]), tensor_arg(a[2]), nullptr, dims, false, float_arg(a[5]), false, true));
  END_HANDLE_TH_ERRORS
}

// the same -> (o, lse2, o's low part or None) and (q, k, v, o, lse2, low part, do, the same 3 numbers) -> (dq, dk, dv): no graph, no padding
PyObject* py_window_forward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 6, 6);
  at::AutoDispatchBelowADInplaceOrView below;
  const Tensor &q = tensor_arg(a[0]), &k = tensor_arg(a[1]), &v = tensor_arg(a[2]);
  const int64_t dims[2] = {window_arg(a[3]), int_arg(a[4])};
  require_gpu(q, k, v);
  check_assert(q.dim() == 4, "q, k and v must have shape [B, heads, L, D]");
  const Tensor q_ = as_rows16(q, group_of(q, k)), k_ = as_rows16(k), v_ = as_rows16(v);
  const Forward f = run_forward(window_spec(q_, k_, v_, dims, float_arg(a[5])), q_, k_, v_, nullptr, false);
  return Py_BuildValue("(NNN)", THPVariable_Wrap(f.o), THPVariable_Wrap(f.lse), THPVariable_Wrap(f.low));
  END_HANDLE_TH_ERRORS
}

PyObject* py_window_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 10, 10);
  at::AutoDispatchBelowADInplaceOrView below;
  const Tensor &q = tensor_arg(a[0]), &k = tensor_arg(a[1]), &v = tensor_arg(a[2]), &o = tensor_arg(a[3]), &lse = tensor_arg(a[4]), &d_o = tensor_arg(a[6]);
  const Tensor low = a[5] == Py_None ? Tensor() : tensor_arg(a[5]).contiguous();
  const int64_t dims[2] = {window_arg(a[7]), int_arg(a[8])};
  require_gpu(q, k, v, o, lse, d_o);
  check_assert(q.dim() == 4, "q, k and v must have shape [B, heads, L, D]");
  const Tensor q_ = as_rows16(q, group_of(q, k)), k_ = as_rows16(k), v_ = as_rows16(v), o_ = as_rows16(o);
  auto g = run_backward(window_spec(q_, k_, v_, dims, float_arg(a[9])), q_, k_, v_, o_, lse.contiguous(), d_o, nullptr, false, low);
  return Py_BuildValue("(NNN)", THPVariable_Wrap(g[0]), THPVariable_Wrap(g[1]), THPVariable_Wrap(g[2]));
  END_HANDLE_TH_ERRORS
}

Axes axes_arg(PyObject* pos, PyObject* tables, PyObject* layout) {
  Axes t;
  if (pos != Py_None) t.pos = tensor_arg(pos);
  PyObject* seq = PySequence_Fast(tables, "tables must be a sequence of cos/sin tables");
  if (seq == nullptr) throw python_error();
  const Py_ssize_t n = PySequence_Fast_GET_SIZE(seq);
  for (Py_ssize_t i = 0; i < n; i++) {
    PyObject* o = PySequence_Fast_GET_ITEM(seq, i);
    if (!THPVariable_Check(o)) {
      Py_DECREF(seq);
      raise_py(PyExc_TypeError, "tables must hold tensors");
    }
    t.tables.push_back(THPVariable_Unpack(o));
  }
  Py_DECREF(seq);
  t.layout = (int)int_arg(layout);
  return t;
}
bool plain_axes(const Axes& t) {
  bool ok = plain_each(t.pos);
  for (const Tensor& x : t.tables) ok = ok && plain(x);
  return ok;
}
PyObject* wrap_pair(const Tensor& q, const Tensor& k) {
  if (!k.defined()) return Py_BuildValue("(NO)", THPVariable_Wrap(q), Py_None);
  return Py_BuildValue("(NN)", THPVariable_Wrap(q), THPVariable_Wrap(k));
}

// (q, k or None, pos, tables, layout number, inverse, mode): mode 0: new tensors, with a graph; 1: new tensors, no graph; 2: in place, no graph; 3: the same
// for any call (0 and 2 take plain ones)
PyObject* py_rope_axes(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 7, 7);
  const Tensor& q = tensor_arg(a[0]);
  const Tensor k = a[1] == Py_None ? Tensor() : tensor_arg(a[1]);
  const Axes t = axes_arg(a[2], a[3], a[4]);
  const bool inverse = bool_arg(a[5]);
  const int64_t mode = int_arg(a[6]);
  if ((mode == 0 || mode == 2) && !(plain_each(q, k) && plain_axes(t))) Py_RETURN_NOTIMPLEMENTED;
  if (mode == 0) {
    const auto out = rope_axes(q, k, t, inverse);
    return wrap_pair(out[0], out[1]);
  }
  if (mode >= 2) {
    require_gpu(q);
    check_written(q, "q");
    if (k.defined()) {
      require_gpu(q, k);
      check_written(k, "k");
      check_two(q, k, "q and k");
    }
    torch::autograd::check_inplace(q, torch::autograd::compute_requires_grad(q));
    if (k.defined()) torch::autograd::check_inplace(k, torch::autograd::compute_requires_grad(k));
    {
      at::AutoDispatchBelowADInplaceOrView below;
      run_axes(q, k, q, k, t, inverse);
    }
    torch::autograd::increment_version(q);
    if (k.defined()) torch::autograd::increment_version(k);
    return PyTuple_Pack(2, a[0], a[1]);
  }
  at::AutoDispatchBelowADInplaceOrView below;
  const auto out = run_axes_new(q, k, t, inverse);
  return wrap_pair(out[0], out[1]);
  END_HANDLE_TH_ERRORS
}

// (k_cache, v_cache, k, v, page_table, seq_len, n_new or None, pos or None, tables or None, layout number, q or None, any call or plain ones only) -> rotated q or None
PyObject* py_paged_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 12, 12);
  const Tensor &kc = tensor_arg(a[0]), &vc = tensor_arg(a[1]), &k = tensor_arg(a[2]), &v = tensor_arg(a[3]), &table = tensor_arg(a[4]), &seq = tensor_arg(a[5]);
  const Tensor n_new = a[6] == Py_None ? Tensor() : tensor_arg(a[6]), q = a[10] == Py_None ? Tensor() : tensor_arg(a[10]);
  const bool rope = a[8] != Py_None;
  Axes t;
  if (rope) t = axes_arg(a[7], a[8], a[9]);
  for (const Tensor* c : {&kc, &vc}) torch::autograd::check_inplace(*c, torch::autograd::compute_requires_grad(*c));
  if (!bool_arg(a[11]) && !(plain(kc, vc, k, v, table, seq) && plain_each(n_new, q) && plain_axes(t))) Py_RETURN_NOTIMPLEMENTED;
  check_assert(k.dim() == 4 && v.dim() == 4 && k.sizes().slice(0, 3) == v.sizes().slice(0, 3), "k and v must have shape [B, heads, T, D], all but D alike");
  check_assert(k.size(1) == kc.size(1) && k.size(3) == kc.size(3) && v.size(3) == vc.size(3), "k and v must match their caches");
  check_assert(k.scalar_type() == kc.scalar_type() && v.scalar_type() == kc.scalar_type(), "k, v and the caches must have one dtype");
  check_assert(!q.defined() || (q.dim() == 4 && q.size(0) == k.size(0) && q.size(2) == k.size(2) && q.size(3) == k.size(3) && q.scalar_type() == k.scalar_type()),
               "q must match k");
  Paged p = paged_args(kc, vc, table, seq, n_new.defined() ? &n_new : nullptr, k.size(0), k.size(2), q.defined() ? q.size(1) : 0);
  require_gpu(kc, k, v);
  if (q.defined()) require_gpu(kc, q);
  check_written(kc, "k_cache");
  check_written(vc, "v_cache");
  check_two(kc, vc, "k_cache and v_cache");
  Tensor q_out;
  if (p.s.B > 0) {
    at::AutoDispatchBelowADInplaceOrView below;
    c10::DeviceGuard guard(kc.device());
    if (q.defined()) q_out = empty(q.sizes(), q.scalar_type(), q);
    dlt_rope_axes_t d;
    if (rope) make_axes(t, k.size(0), k.size(2), kc, d);
    check_rc(dlt_paged_append(k.const_data_ptr(), st(k), v.const_data_ptr(), st(v), q.defined() ? q.const_data_ptr() : nullptr, q.defined() ? st(q) : nullptr,
                              q.defined() ? q_out.mutable_data_ptr() : nullptr, q.defined() ? st(q_out) : nullptr, kc.mutable_data_ptr(), st(kc),
                              vc.mutable_data_ptr(), st(vc), p.table, p.ts, p.seq, p.n_new, rope ? &d : nullptr, &p.s, stream_of(kc)));
  } else if (q.defined()) {
    q_out = empty(q.sizes(), q.scalar_type(), q);
  }
  torch::autograd::increment_version(kc);
  torch::autograd::increment_version(vc);
  if (!q_out.defined()) Py_RETURN_NONE;
  return THPVariable_Wrap(q_out);
  END_HANDLE_TH_ERRORS
}

// (q, k_cache, v_cache, page_table, seq_len, window or None, n_sink, scale, n_new or None, any call or plain ones only) -> o, no graph
PyObject* py_paged_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 10, 10);
  const Tensor &q0 = tensor_arg(a[0]), &kc = tensor_arg(a[1]), &vc = tensor_arg(a[2]), &table = tensor_arg(a[3]), &seq = tensor_arg(a[4]);
  const Tensor n_new = a[8] == Py_None ? Tensor() : tensor_arg(a[8]);
  if (!bool_arg(a[9]) && !(plain(q0, kc, vc, table, seq) && plain_each(n_new))) Py_RETURN_NOTIMPLEMENTED;
  at::AutoDispatchBelowADInplaceOrView below;
  check_assert(q0.dim() == 4 && q0.size(3) == kc.size(-1) && q0.scalar_type() == kc.scalar_type(), "q must have shape [B, heads, T, D] and match the cache");
  Paged p = paged_args(kc, vc, table, seq, n_new.defined() ? &n_new : nullptr, q0.size(0), q0.size(2), q0.size(1));
  p.s.window = window_arg(a[5]);
  p.s.n_sink = (int32_t)int_arg(a[6]);
  p.s.sm_scale = (float)float_arg(a[7]);
  require_gpu(kc, q0);
  require(rows16(kc) && rows16(vc), PyExc_ValueError, "rows of the caches must be contiguous and start at multiples of 16 bytes");
  c10::DeviceGuard guard(kc.device());
  Tensor o = empty({q0.size(0), q0.size(1), q0.size(2), vc.size(3)}, q0.scalar_type(), q0);
  if (o.numel() == 0) return THPVariable_Wrap(o);
  const Tensor q = as_rows16(q0, group_of(q0, kc));
  Workspace ws;
  check_rc(dlt_paged_workspace(&p.s, &ws.bytes));
  if (ws.bytes > 0) {
    ws.t = empty({ws.bytes / 4}, at::kFloat, q);
    ws.ptr = ws.t.mutable_data_ptr();
  }
  check_rc(dlt_paged_attn(q.const_data_ptr(), st16(q).data(), kc.const_data_ptr(), st16(kc).data(), vc.const_data_ptr(), st16(vc).data(), o.mutable_data_ptr(),
                          st16(o).data(), p.table, p.ts, p.seq, p.n_new, &p.s, ws.ptr, ws.bytes, stream_of(q)));
  return THPVariable_Wrap(o);
  END_HANDLE_TH_ERRORS
}

// Caches of 8-bit numbers [pages, heads, page, D] and their scales [pages, heads, page / block]
dlt_scales8_t scales_of(const Tensor& kc, const Tensor& vc, const Tensor& ks, const Tensor& vs) {
  require((kc.scalar_type() == at::kFloat8_e4m3fn || kc.scalar_type() == at::kChar) && vc.scalar_type() == kc.scalar_type(), PyExc_TypeError,
          "caches must be float8_e4m3fn or int8, both alike");
  require(ks.scalar_type() == at::kFloat8_e8m0fnu && vs.scalar_type() == at::kFloat8_e8m0fnu, PyExc_TypeError, "scales must be float8_e8m0fnu");
  check_assert(kc.dim() == 4 && vc.dim() == 4, "caches must have shape [pages, heads, page, D], all but D alike");
  check_assert(ks.dim() == 3 && vs.dim() == 3 && ks.sizes() == vs.sizes() && ks.sizes().slice(0, 2) == kc.sizes().slice(0, 2), "scales must have shape [pages, heads, blocks of a page]");
  require(ks.size(2) > 0 && kc.size(2) % ks.size(2) == 0, PyExc_ValueError, "the blocks of a page must have one size");
  require_gpu(kc, ks, vs);
  dlt_scales8_t x{};
  x.format = kc.scalar_type() == at::kChar ? DLT_INT8 : DLT_FP8_E4M3;
  x.block = (int32_t)(kc.size(2) / ks.size(2));
  x.k_scale = const_cast<void*>(ks.const_data_ptr());
  x.v_scale = const_cast<void*>(vs.const_data_ptr());
  for (int i = 0; i < 3; i++) {
    x.k_strides[i] = ks.size(i) == 1 ? 0 : ks.stride(i);
    x.v_strides[i] = vs.size(i) == 1 ? 0 : vs.stride(i);
  }
  return x;
}
// rows of 8-bit numbers that the kernels can read in 8-byte pieces
bool rows8(const Tensor& x) {
  bool ok = (x.stride(3) == 1 || x.size(3) == 1) && (uintptr_t)x.const_data_ptr() % 8 == 0;
  for (int i = 0; i < 3; i++) ok = ok && (x.size(i) == 1 || (x.stride(i) % 8 == 0 && x.stride(i) >= 0));
  return ok;
}
// rows in 16-byte pieces, else a copy
Tensor as_pieces(const Tensor& x) {
  if (x.dim() != 4 || x.numel() == 0) return x;
  const int64_t n = 16 / (int64_t)x.element_size();
  bool ok = (x.stride(3) == 1 || x.size(3) == 1) && (uintptr_t)x.const_data_ptr() % 16 == 0;
  for (int i = 0; i < 3; i++) ok = ok && (x.size(i) == 1 || x.stride(i) % n == 0);
  return ok ? x : x.clone(at::MemoryFormat::Contiguous);
}

// (k_cache, v_cache, k_scale, v_scale, k, v, page_table, seq_len, n_new or None, pos or None, tables or None, layout number, q or None, any call or plain ones only) -> rotated q or None
PyObject* py_paged8_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 14, 14);
  const Tensor &kc = tensor_arg(a[0]), &vc = tensor_arg(a[1]), &ks = tensor_arg(a[2]), &vs = tensor_arg(a[3]), &k0 = tensor_arg(a[4]), &v0 = tensor_arg(a[5]), &table = tensor_arg(a[6]),
               &seq = tensor_arg(a[7]);
  const Tensor n_new = a[8] == Py_None ? Tensor() : tensor_arg(a[8]), q0 = a[12] == Py_None ? Tensor() : tensor_arg(a[12]);
  const bool rope = a[10] != Py_None;
  Axes t;
  if (rope) t = axes_arg(a[9], a[10], a[11]);
  for (const Tensor* c : {&kc, &vc, &ks, &vs}) torch::autograd::check_inplace(*c, torch::autograd::compute_requires_grad(*c));
  if (!bool_arg(a[13]) && !(plain(kc, vc, ks, vs, k0, v0, table, seq) && plain_each(n_new, q0) && plain_axes(t))) Py_RETURN_NOTIMPLEMENTED;
  check_assert(k0.dim() == 4 && v0.dim() == 4 && k0.sizes().slice(0, 3) == v0.sizes().slice(0, 3), "k and v must have shape [B, heads, T, D], all but D alike");
  dlt_scales8_t scales = scales_of(kc, vc, ks, vs);
  check_assert(k0.size(1) == kc.size(1) && k0.size(3) == kc.size(3) && v0.size(3) == vc.size(3), "k and v must match their caches");
  check_assert(k0.scalar_type() == v0.scalar_type(), "k and v must have one dtype");
  check_assert(!q0.defined() || (q0.dim() == 4 && q0.size(0) == k0.size(0) && q0.size(2) == k0.size(2) && q0.size(3) == k0.size(3) && q0.scalar_type() == k0.scalar_type()),
               "q must match k");
  Paged p = paged_args(kc, vc, table, seq, n_new.defined() ? &n_new : nullptr, k0.size(0), k0.size(2), q0.defined() ? q0.size(1) : 0, dtype_code(k0));
  require_gpu(kc, k0, v0);
  if (q0.defined()) require_gpu(kc, q0);
  require(rows8(kc) && rows8(vc), PyExc_ValueError, "rows of the caches must be contiguous and start at multiples of 8 bytes");
  const std::pair<const Tensor*, const char*> written[] = {{&kc, "k_cache"}, {&vc, "v_cache"}, {&ks, "k_scale"}, {&vs, "v_scale"}};
  for (const auto& w : written) check_written(*w.first, w.second);
  for (int i = 0; i < 4; i++)
    for (int j = i + 1; j < 4; j++) check_two(*written[i].first, *written[j].first, "the caches and their scales");
  Tensor q_out;
  if (q0.defined()) {
    c10::DeviceGuard guard(kc.device());
    q_out = empty(q0.sizes(), q0.scalar_type(), q0);
  }
  if (p.s.B > 0) {
    at::AutoDispatchBelowADInplaceOrView below;
    c10::DeviceGuard guard(kc.device());
    const Tensor k = as_pieces(k0), v = as_pieces(v0), q = q0.defined() ? as_pieces(q0) : q0;
    dlt_rope_axes_t d;
    if (rope) make_axes(t, k.size(0), k.size(2), kc, d);
    check_rc(dlt_paged8_append(k.const_data_ptr(), st16(k).data(), v.const_data_ptr(), st16(v).data(), q.defined() ? q.const_data_ptr() : nullptr,
                               q.defined() ? st16(q).data() : nullptr, q.defined() ? q_out.mutable_data_ptr() : nullptr, q.defined() ? st16(q_out).data() : nullptr,
                               kc.mutable_data_ptr(), st16(kc).data(), vc.mutable_data_ptr(), st16(vc).data(), &scales, p.table, p.ts, p.seq, p.n_new, rope ? &d : nullptr, &p.s,
                               stream_of(kc)));
  }
  for (const auto& w : written) torch::autograd::increment_version(*w.first);
  if (!q_out.defined()) Py_RETURN_NONE;
  return THPVariable_Wrap(q_out);
  END_HANDLE_TH_ERRORS
}

// (q, k_cache, v_cache, k_scale, v_scale, page_table, seq_len, window or None, n_sink, scale, n_new or None, any call or plain ones only) -> o, no graph
PyObject* py_paged8_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 12, 12);
  const Tensor &q0 = tensor_arg(a[0]), &kc = tensor_arg(a[1]), &vc = tensor_arg(a[2]), &ks = tensor_arg(a[3]), &vs = tensor_arg(a[4]), &table = tensor_arg(a[5]), &seq = tensor_arg(a[6]);
  const Tensor n_new = a[10] == Py_None ? Tensor() : tensor_arg(a[10]);
  if (!bool_arg(a[11]) && !(plain(q0, kc, vc, ks, vs, table, seq) && plain_each(n_new))) Py_RETURN_NOTIMPLEMENTED;
  at::AutoDispatchBelowADInplaceOrView below;
  const dlt_scales8_t scales = scales_of(kc, vc, ks, vs);
  check_assert(q0.dim() == 4 && q0.size(3) == kc.size(3), "q must have shape [B, heads, T, D] and match the cache");
  Paged p = paged_args(kc, vc, table, seq, n_new.defined() ? &n_new : nullptr, q0.size(0), q0.size(2), q0.size(1), dtype_code(q0));
  p.s.window = window_arg(a[7]);
  p.s.n_sink = (int32_t)int_arg(a[8]);
  p.s.sm_scale = (float)float_arg(a[9]);
  require_gpu(kc, q0);
  require(rows8(kc) && rows8(vc), PyExc_ValueError, "rows of the caches must be contiguous and start at multiples of 8 bytes");
  c10::DeviceGuard guard(kc.device());
  Tensor o = empty({q0.size(0), q0.size(1), q0.size(2), vc.size(3)}, q0.scalar_type(), q0);
  if (o.numel() == 0) return THPVariable_Wrap(o);
  const Tensor q = as_rows16(q0, group_of(q0, kc));
  Workspace ws;
  check_rc(dlt_paged8_workspace(&p.s, &scales, &ws.bytes));
  if (ws.bytes > 0) {
    ws.t = empty({ws.bytes / 4}, at::kFloat, q);
    ws.ptr = ws.t.mutable_data_ptr();
  }
  check_rc(dlt_paged8_attn(q.const_data_ptr(), st16(q).data(), kc.const_data_ptr(), st16(kc).data(), vc.const_data_ptr(), st16(vc).data(), &scales, o.mutable_data_ptr(),
                           st16(o).data(), p.table, p.ts, p.seq, p.n_new, &p.s, ws.ptr, ws.bytes, stream_of(q)));
  return THPVariable_Wrap(o);
  END_HANDLE_TH_ERRORS
}

// (page_table, seq_len, want, pool, page, n_tokens or None, any call or plain ones only) -> (n_new, slots or None)
PyObject* py_page_assign(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 7, 7);
  const Tensor &table = tensor_arg(a[0]), &seq = tensor_arg(a[1]), &want = tensor_arg(a[2]), &pool = tensor_arg(a[3]);
  if (!bool_arg(a[6]) && !plain(table, seq, want, pool)) Py_RETURN_NOTIMPLEMENTED;
  const int64_t page = int_arg(a[4]), T = a[5] == Py_None ? -1 : int_arg(a[5]);
  auto ints = [](const Tensor& x) { return x.scalar_type() == at::kInt && x.dim() == 1 && (x.size(0) <= 1 || x.stride(0) == 1); };
  require(table.scalar_type() == at::kInt && table.dim() == 2 && (table.size(1) <= 1 || table.stride(1) == 1), PyExc_TypeError,
          "page_table must be an int32 tensor [B, pages of a sequence] with contiguous rows");
  require(ints(seq) && ints(want), PyExc_TypeError, "seq_len and want must be contiguous 1-D int32 tensors");
  require(ints(pool) && pool.size(0) > 2, PyExc_TypeError, "pool must be a contiguous 1-D int32 tensor [2 + pages]");
  const int64_t B = table.size(0);
  check_assert(seq.size(0) == B && want.size(0) == B, "page_table, seq_len and want must have a row for every request");
  require(T >= 0 || a[5] == Py_None, PyExc_ValueError, "n_tokens must not be negative");
  require(page > 0 && table.size(1) > 0, PyExc_ValueError, "pages need a token, and the table a column");
  check_assert(B <= INT32_MAX && table.size(1) <= INT32_MAX && pool.size(0) <= INT32_MAX, "too many requests or pages");
  require_gpu(table, seq, want, pool);
  check_written(table, "page_table");
  check_written(seq, "seq_len");
  check_two(table, seq, "page_table and seq_len");
  check_two(table, pool, "page_table and pool");
  check_two(seq, pool, "seq_len and pool");
  for (const Tensor* x : {&table, &seq, &pool}) require(!meet(want, *x), PyExc_RuntimeError, "want shares memory with a tensor that is written");
  Tensor n_new, slots;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    c10::DeviceGuard guard(table.device());
    n_new = empty({B}, at::kInt, table);
    if (a[5] != Py_None) slots = empty({B, T}, at::kInt, table);
    check_rc(dlt_page_assign(table.mutable_data_ptr<int32_t>(), table.size(0) > 1 ? table.stride(0) : table.size(1), seq.mutable_data_ptr<int32_t>(), want.const_data_ptr<int32_t>(),
                             pool.mutable_data_ptr<int32_t>(), (int32_t)B, (int32_t)table.size(1), (int32_t)page, (int32_t)(pool.size(0) - 2), (int32_t)T,
                             n_new.mutable_data_ptr<int32_t>(), slots.defined() && slots.numel() > 0 ? slots.mutable_data_ptr<int32_t>() : nullptr, stream_of(table)));
  }
  for (const Tensor* x : {&table, &seq, &pool}) torch::autograd::increment_version(*x);
  if (!slots.defined()) return Py_BuildValue("(NO)", THPVariable_Wrap(n_new), Py_None);
  return Py_BuildValue("(NN)", THPVariable_Wrap(n_new), THPVariable_Wrap(slots));
  END_HANDLE_TH_ERRORS
}

// (x[B', N, C], idx, row, col): rotated in place, returned
PyObject* py_rope_apply(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 4, 4);
  const Tensor& x = tensor_arg(a[0]);
  if (!plain(x, tensor_arg(a[1]), tensor_arg(a[2]), tensor_arg(a[3]))) Py_RETURN_NOTIMPLEMENTED;
  if (x.dim() != 3) raise_py(PyExc_ValueError, "x must have shape [B', N, C]");
  Rows r;
  rows_of(x, r);
  rope_apply(x, r, tensor_arg(a[1]), tensor_arg(a[2]), tensor_arg(a[3]));
  Py_INCREF(a[0]);
  return a[0];
  END_HANDLE_TH_ERRORS
}

// (x[B, H, N, C], idx, row, col): rotated in place where B and H are one run of rows, else a rotated copy
PyObject* py_rope_heads(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 4, 4);
  const Tensor& x = tensor_arg(a[0]);
  if (!plain(x, tensor_arg(a[1]), tensor_arg(a[2]), tensor_arg(a[3]))) Py_RETURN_NOTIMPLEMENTED;
  if (x.dim() != 4) raise_py(PyExc_ValueError, "x must have shape [B, H, N, C]");
  Rows r;
  if (C10_LIKELY(rows_of(x, r))) {
    rope_apply(x, r, tensor_arg(a[1]), tensor_arg(a[2]), tensor_arg(a[3]));
    Py_INCREF(a[0]);
    return a[0];
  }
  Tensor y = x.reshape({-1, x.size(2), x.size(3)});
  rows_of(y, r);
  rope_apply(y, r, tensor_arg(a[1]), tensor_arg(a[2]), tensor_arg(a[3]));
  return THPVariable_Wrap(y.reshape(x.sizes()));
  END_HANDLE_TH_ERRORS
}

// (x[B', N, C], idx, row, col, inverse): in place, no graph
PyObject* py_rope_inplace(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 5, 5);
  at::AutoDispatchBelowADInplaceOrView below;
  const Tensor &x = tensor_arg(a[0]), &idx = tensor_arg(a[1]), &row = tensor_arg(a[2]), &col = tensor_arg(a[3]);
  require_gpu(x, idx, row, col);
  if (x.dim() != 3) raise_py(PyExc_ValueError, "x must have shape [B', N, C]");
  Rows r;
  rows_of(x, r);
  rotate_inplace(x, r, make_rope(idx, row, col), bool_arg(a[4]));
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// (q, k, idx, row, col, inverse): both in place with one launch, no graph
PyObject* py_rope_pair(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 6, 6);
  at::AutoDispatchBelowADInplaceOrView below;
  const Tensor &q = tensor_arg(a[0]), &k = tensor_arg(a[1]), &idx = tensor_arg(a[2]), &row = tensor_arg(a[3]), &col = tensor_arg(a[4]);
  require_gpu(q, k, idx, row, col);
  check_assert(q.dim() >= 2 && k.dim() >= 2 && q.size(-2) == k.size(-2) && q.size(-1) == k.size(-1) && q.scalar_type() == k.scalar_type(),
               "q and k must have one token count, head dim and dtype");
  check_assert(idx.dim() != 1 || idx.size(0) >= q.size(-2), "idx must have an entry for every token");
  Rows rq, rk;
  require(rows_of(q, rq) && rows_of(k, rk), PyExc_RuntimeError, "q and k must be viewable as [rows, N, C] (batch and head dims in one run)");
  const Rope rope = make_rope(idx, row, col);
  c10::DeviceGuard guard(q.device());
  check_rc(dlt_rope2d_pair(q.mutable_data_ptr(), rq.s, rq.nb, k.mutable_data_ptr(), rk.s, rk.nb, q.size(-2), q.size(-1), &rope.d, bool_arg(a[5]),
                           dtype_code(q), stream_of(q)));
  return PyTuple_Pack(2, a[0], a[1]);
  END_HANDLE_TH_ERRORS
}

// (dk, dv, dtype-carrying tensor, b_size) -> None or (dk, dv) to pad to; b_size -1: flash
PyObject* py_pad_plan(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 4, 4);
  const int64_t dk = int_arg(a[0]), dv = int_arg(a[1]), b = int_arg(a[3]);
  const at::ScalarType dt = tensor_arg(a[2]).scalar_type();
  const Pad p = b < 0 ? flash_pad(dk, dv, dt) : swa_pad(dk, dv, dt, b);
  if (p.dk == dk && p.dv == dv) Py_RETURN_NONE;
  return Py_BuildValue("(LL)", (long long)p.dk, (long long)p.dv);
  END_HANDLE_TH_ERRORS
}

#define DLT_FN(name) {#name, (PyCFunction)(void (*)(void))py_##name, METH_FASTCALL, nullptr}
PyMethodDef METHODS[] = {DLT_FN(tiled_swa), DLT_FN(tiled_swa_fwd), DLT_FN(tiled_swa_rope), DLT_FN(tiled_swa_image), DLT_FN(flash), DLT_FN(swa_forward),
                         DLT_FN(swa_backward), DLT_FN(image_forward), DLT_FN(image_backward), DLT_FN(flash_forward), DLT_FN(flash_backward), DLT_FN(rope_apply), DLT_FN(rope_heads), DLT_FN(rope_inplace), DLT_FN(rope_pair),
                         DLT_FN(pad_plan), DLT_FN(window), DLT_FN(window_forward), DLT_FN(window_backward), DLT_FN(rope_axes), DLT_FN(paged_append), DLT_FN(paged_attention), DLT_FN(page_assign), DLT_FN(paged8_append), DLT_FN(paged8_attention),
                         {nullptr, nullptr, 0, nullptr}};
#undef DLT_FN

PyModuleDef MODULE = {PyModuleDef_HEAD_INIT, "_dlt_torch", "torch binding of libdlt_hip.so", -1, METHODS, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__dlt_torch() {
  PyObject* lib = PyImport_ImportModule("dl_templates_amd._lib");
  if (lib == nullptr) return nullptr;
  g_dlt_error = PyObject_GetAttrString(lib, "DltError");
  Py_DECREF(lib);
  if (g_dlt_error == nullptr) return nullptr;
  return PyModule_Create(&MODULE);
}
