// Python binding of the window / paged attention operators: argument checks
// on torch tensors, output allocation, and the call into libgpo.so
// (include/gpo.h).  It exists for the calls' latency: a single token's append
// is a 4 us kernel behind a 5 us launch, and the same checks and records took
// 13 us in Python.
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/extension.h>

#include <algorithm>
#include <cstdint>
#include <cstdio>
#include <map>
#include <mutex>
#include <string>

#include "gpo.h"

namespace {

using at::Tensor;
namespace py = pybind11;

py::object g_refused;  // KernelBuildError(message, log=...)

[[noreturn]] void refuse(const std::string& message, const std::string& log) {
  py::object e = g_refused(message, py::arg("log") = log);
  PyErr_SetObject(g_refused.ptr(), e.ptr());
  throw py::error_already_set();
}
[[noreturn]] void refuse(const std::string& message) { refuse(message, message); }

std::string shape_of(at::IntArrayRef s) {
  std::string r = "(";
  for (size_t i = 0; i < s.size(); ++i) r += (i ? ", " : "") + std::to_string(s[i]);
  return r + ")";
}
const char* type_name(at::ScalarType t) {
  switch (t) {
    case at::kHalf: return "torch.float16";
    case at::kBFloat16: return "torch.bfloat16";
    case at::kFloat: return "torch.float32";
    case at::kInt: return "torch.int32";
    default: return c10::toString(t);
  }
}

void check(const char* name, const Tensor& t, int64_t dims, at::ScalarType type,
           const c10::Device& device) {
  if (!t.is_cuda()) refuse(std::string(name) + " must be a CUDA tensor");
  if (t.dim() != dims)
    refuse(std::string(name) + " must have " + std::to_string(dims) + " dimensions, got " +
           shape_of(t.sizes()));
  if (t.scalar_type() != type)
    refuse(std::string(name) + " must be " + type_name(type) + ", got " +
           type_name(t.scalar_type()));
  if (t.device() != device)
    refuse(std::string(name) + " is on " + t.device().str() + ", expected " + device.str());
}

void check_shape(const char* name, const Tensor& t, at::IntArrayRef want) {
  if (t.sizes() != want)
    refuse(std::string(name) + " has shape " + shape_of(t.sizes()) + ", expected " +
           shape_of(want));
}

// A size as the library's records hold it.
int32_t size32(const char* name, int64_t n) {
  if (n < 0 || n > INT32_MAX) refuse(std::string(name) + " is out of range: " + std::to_string(n));
  return static_cast<int32_t>(n);
}

int dtype_id(at::ScalarType t) { return t == at::kBFloat16 ? GPO_BFLOAT16 : GPO_FLOAT16; }

// Whether the kernels can address the tensor's rows where they are.
bool in_place(const Tensor& t) {
  if (t.numel() == 0) return true;
  const auto n = t.sizes(), s = t.strides();
  const size_t last = n.size() - 1;
  if ((s[last] != 1 && n[last] != 1) || (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15u))
    return false;
  for (size_t i = 0; i < last; ++i)
    if (n[i] > 1 && (s[i] & 7)) return false;
  return true;
}

// The tensor, or a copy where its rows cannot be read in place: rows that are
// not contiguous, or a start or stride off the 16-byte grid.
Tensor readable(const Tensor& t) {
  return in_place(t) ? t : t.clone(at::MemoryFormat::Contiguous);
}

void check_written(const char* name, const Tensor& t, at::IntArrayRef shape, at::ScalarType type,
                   const c10::Device& device) {
  check(name, t, static_cast<int64_t>(shape.size()), type, device);
  if (t.sizes() != shape || !(type == at::kFloat ? t.is_contiguous() : in_place(t)))
    refuse(std::string(name) + " must have shape " + shape_of(shape) +
           ", its rows contiguous and 16-byte aligned");
}

gpo_heads heads4(const Tensor& t) {
  return gpo_heads{t.data_ptr(), t.stride(0), t.stride(1), t.stride(2)};
}
gpo_heads heads3(const Tensor& t) { return gpo_heads{t.data_ptr(), 0, t.stride(0), t.stride(1)}; }

void set_mask(c10::optional<int64_t> window, int64_t sinks, c10::optional<double> scale,
              int64_t& w, int64_t& s, float& f) {
  if (window && *window < 1)
    refuse("window must be at least 1 (or None), got " + std::to_string(*window));
  if (sinks < 0) refuse("sinks must not be negative, got " + std::to_string(sinks));
  // as a float: what rounds to 0 would ask for the default
  if (scale && !(static_cast<float>(*scale) > 0.f)) {
    char text[64];
    snprintf(text, sizeof(text), "scale must be positive (2^-126 at least), got %g", *scale);
    refuse(text);
  }
  w = window ? *window : 0;
  s = sinks;
  f = scale ? static_cast<float>(*scale) : 0.f;
}

typedef gpo_status (*WindowFn)(const gpo_window_args*, void*, char*, size_t);
typedef gpo_status (*PagedFn)(const gpo_paged_args*, void*, char*, size_t);

void raise_status(const char* name, gpo_status s, const char* why) {
  const std::string text = std::string(name) + ": " + gpo_status_name(s) + ": " + why;
  if (s == GPO_BAD_ARGS || s == GPO_BAD_CONFIG) refuse(text, why);
  throw std::runtime_error(text);
}

template <typename F, typename A>
void launch(const char* name, F fn, const A& args, const c10::Device& device) {
  char log[256];
  c10::cuda::OptionalCUDAGuard guard;
  if (c10::cuda::current_device() != device.index()) guard.set_device(device);
  const gpo_status s =
      fn(&args, c10::cuda::getCurrentCUDAStream(device.index()).stream(), log, sizeof(log));
  if (s != GPO_OK) raise_status(name, s, log);
}

// ------------------------------------------------------------------ window
gpo_window_args window_args(const Tensor& q, const Tensor& k, const Tensor& v,
                            c10::optional<int64_t> window, int64_t sinks,
                            c10::optional<double> scale) {
  const auto type = q.scalar_type();
  if (type != at::kHalf && type != at::kBFloat16)
    refuse("q must be a float16 or bfloat16 CUDA tensor");
  const auto device = q.device();
  check("q", q, 4, type, device);
  check("k", k, 4, type, device);
  check("v", v, 4, type, device);
  if (k.sizes() != v.sizes() || k.size(0) != q.size(0) || k.size(3) != q.size(3))
    refuse("q " + shape_of(q.sizes()) + ", k " + shape_of(k.sizes()) + " and v " +
           shape_of(v.sizes()) + " do not belong together");
  gpo_window_args a{};
  a.dtype = dtype_id(type);
  a.head_dim = size32("head_dim", q.size(3));
  a.heads_q = size32("heads_q", q.size(2));
  a.heads_kv = size32("heads_kv", k.size(2));
  a.batch = q.size(0);
  a.q_len = q.size(1);
  a.kv_len = k.size(1);
  set_mask(window, sinks, scale, a.window, a.sinks, a.scale);
  return a;
}

std::pair<Tensor, Tensor> window_forward(const Tensor& q0, const Tensor& k0, const Tensor& v0,
                                         c10::optional<int64_t> window, int64_t sinks,
                                         c10::optional<double> scale,
                                         c10::optional<Tensor> out0, c10::optional<Tensor> lse0) {
  gpo_window_args a = window_args(q0, k0, v0, window, sinks, scale);
  const Tensor q = readable(q0), k = readable(k0), v = readable(v0);
  const auto rows = q.sizes().slice(0, 3);
  if (out0) check_written("out", *out0, q.sizes(), q.scalar_type(), q.device());
  if (lse0) check_written("lse", *lse0, rows, at::kFloat, q.device());
  Tensor out = out0 ? *out0 : at::empty(q.sizes(), q.options());
  Tensor lse = lse0 ? *lse0 : at::empty(rows, q.options().dtype(at::kFloat));
  a.q = heads4(q);
  a.k = heads4(k);
  a.v = heads4(v);
  a.out = heads4(out);
  a.lse = static_cast<float*>(lse.data_ptr());
  launch("gpo_window_attention", gpo_window_attention, a, q.device());
  return {out, lse};
}

std::tuple<Tensor, Tensor, Tensor> window_backward(
    const Tensor& dout0, const Tensor& q0, const Tensor& k0, const Tensor& v0, const Tensor& out0,
    const Tensor& lse0, c10::optional<int64_t> window, int64_t sinks, c10::optional<double> scale,
    c10::optional<std::tuple<Tensor, Tensor, Tensor>> grads) {
  gpo_window_args a = window_args(q0, k0, v0, window, sinks, scale);
  const auto type = q0.scalar_type();
  const auto device = q0.device();
  const auto rows = q0.sizes().slice(0, 3);
  check("out", out0, 4, type, device);
  check_shape("out", out0, q0.sizes());
  check("dout", dout0, 4, type, device);
  check_shape("dout", dout0, q0.sizes());
  check("lse", lse0, 3, at::kFloat, device);
  check_shape("lse", lse0, rows);
  const Tensor q = readable(q0), k = readable(k0), v = readable(v0), out = readable(out0),
               dout = readable(dout0), lse = lse0.contiguous();
  Tensor dq, dk, dv;
  if (grads) {
    std::tie(dq, dk, dv) = *grads;
    check_written("dq", dq, q.sizes(), type, device);
    check_written("dk", dk, k.sizes(), type, device);
    check_written("dv", dv, k.sizes(), type, device);
  } else {
    dq = at::empty(q.sizes(), q.options());
    dk = at::empty(k.sizes(), q.options());
    dv = at::empty(k.sizes(), q.options());
  }
  a.q = heads4(q);
  a.k = heads4(k);
  a.v = heads4(v);
  a.out = heads4(out);
  a.dout = heads4(dout);
  a.dq = heads4(dq);
  a.dk = heads4(dk);
  a.dv = heads4(dv);
  a.lse = static_cast<float*>(lse.data_ptr());
  char log[256];
  const gpo_status s = gpo_window_workspace(&a, &a.workspace_bytes, log, sizeof(log));
  if (s != GPO_OK) raise_status("gpo_window_workspace", s, log);
  Tensor work;
  if (a.workspace_bytes) {
    work = at::empty({static_cast<int64_t>(a.workspace_bytes)}, q.options().dtype(at::kByte));
    a.workspace = work.data_ptr();
  }
  launch("gpo_window_attention_grad", gpo_window_attention_grad, a, device);
  return {dq, dk, dv};
}

// ------------------------------------------------------------------- paged
// The stream of a device that plans are made on: one for all, so that a plan
// takes up the memory that another has given back, and not one of the pool,
// where other work may be queued.
c10::cuda::CUDAStream plan_stream(c10::DeviceIndex device) {
  static std::mutex mutex;
  static std::map<c10::DeviceIndex, cudaStream_t> streams;
  const std::lock_guard<std::mutex> lock(mutex);
  cudaStream_t& s = streams[device];
  if (!s) C10_CUDA_CHECK(cudaStreamCreateWithFlags(&s, cudaStreamNonBlocking));
  return c10::cuda::getStreamFromExternal(s, device);
}

constexpr int64_t kMostTokens = 1ll << 30;  // of a call (gpo.h)

struct Plan {
  gpo_paged_args args{};
  at::ScalarType type;
  c10::Device device{c10::kCPU};
  int64_t max_seqs;
  Tensor work;
  mutable c10::optional<c10::cuda::CUDAStream> held_by;  // the last call's stream

  Plan(int64_t heads_q, int64_t heads_kv, int64_t head_dim, int64_t page_size, int64_t max_seqs_,
       int64_t max_q, at::ScalarType type_, c10::optional<int64_t> window, int64_t sinks,
       c10::optional<double> scale, c10::Device device_)
      : type(type_), device(device_), max_seqs(max_seqs_) {
    if (type != at::kHalf && type != at::kBFloat16)
      refuse(std::string("dtype must be float16 or bfloat16, got ") + type_name(type));
    if (max_seqs < 1 || max_q < 1) refuse("max_seqs and max_q must be at least 1");
    args.dtype = dtype_id(type);
    args.head_dim = size32("head_dim", head_dim);
    args.heads_q = size32("heads_q", heads_q);
    args.heads_kv = size32("heads_kv", heads_kv);
    args.page_size = page_size;
    args.max_q = max_q;
    args.num_seqs = max_seqs;
    // of all sequences at their longest, or what the library takes in one call
    args.tokens = std::min<int64_t>(kMostTokens / max_seqs, max_q) * max_seqs;
    set_mask(window, sinks, scale, args.window, args.sinks, args.scale);
    char log[256];
    const gpo_status s = gpo_paged_workspace(&args, &args.workspace_bytes, log, sizeof(log));
    if (s != GPO_OK) raise_status("gpo_paged_workspace", s, log);
    make_workspace();
    args.workspace = work.data_ptr();
  }

  // The workspace is zero before the plan is handed out, whichever stream
  // calls it first.  It is made on the plans' own stream, which alone is
  // waited for; in a capture the zeroing becomes a part of the graph.
  void make_workspace() {
    const auto bytes = static_cast<int64_t>(args.workspace_bytes);
    const auto options = at::TensorOptions().dtype(at::kByte).device(device);
    const c10::cuda::CUDAGuard on(device);
    if (c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None) {
      work = at::zeros({bytes}, options);
      return;
    }
    const auto own = plan_stream(device.index());
    const c10::cuda::CUDAStreamGuard guard(own);
    work = at::zeros({bytes}, options);
    own.synchronize();
  }

  // Keeps the workspace from being handed on, if the plan is dropped, before
  // the calls on this stream are done.
  void hold_workspace() const {
    const auto stream = c10::cuda::getCurrentCUDAStream(device.index());
    if (held_by == stream) return;
    c10::cuda::CUDACachingAllocator::recordStream(work.storage().data_ptr(), stream);
    held_by = stream;
  }

  gpo_paged_args fill(int64_t rows, const Tensor& k_pages, const Tensor& v_pages,
                      const Tensor& table, const Tensor& q_start, const Tensor& kv_len) const {
    gpo_paged_args a = args;
    const int64_t page[3] = {a.page_size, a.heads_kv, a.head_dim};
    for (int i = 0; i < 2; ++i) {
      const char* name = i ? "v_pages" : "k_pages";
      const Tensor& t = i ? v_pages : k_pages;
      check(name, t, 4, type, device);
      if (t.sizes().slice(1) != at::IntArrayRef(page, 3))
        refuse(std::string(name) + " has shape " + shape_of(t.sizes()) + ", expected (pages, " +
               shape_of(at::IntArrayRef(page, 3)).substr(1));
      if (!in_place(t))
        refuse(std::string(name) + ": rows must be contiguous and 16-byte aligned");
    }
    if (k_pages.size(0) != v_pages.size(0))
      refuse("k_pages and v_pages have different numbers of pages");
    check("page_table", table, 2, at::kInt, device);
    check("q_start", q_start, 1, at::kInt, device);
    check("kv_len", kv_len, 1, at::kInt, device);
    const int64_t seqs = table.size(0), width = table.size(1);
    if (seqs > max_seqs || q_start.size(0) != seqs + 1 || kv_len.size(0) != seqs)
      refuse(std::to_string(seqs) + " sequences in page_table, " +
             std::to_string(q_start.size(0) - 1) + " in q_start, " +
             std::to_string(kv_len.size(0)) + " in kv_len; at most " + std::to_string(max_seqs));
    if ((width > 1 && table.stride(1) != 1) || !q_start.is_contiguous() ||
        !kv_len.is_contiguous())
      refuse("page_table rows, q_start and kv_len must be contiguous");
    a.num_seqs = seqs;
    a.tokens = rows;
    a.num_pages = k_pages.size(0);
    a.table_width = width;
    a.table_stride = table.stride(0);
    a.page_table = static_cast<const int32_t*>(table.data_ptr());
    a.q_start = static_cast<const int32_t*>(q_start.data_ptr());
    a.kv_len = static_cast<const int32_t*>(kv_len.data_ptr());
    a.k_pages = heads4(k_pages);
    a.v_pages = heads4(v_pages);
    return a;
  }

  void append(const Tensor& k0, const Tensor& v0, const Tensor& k_pages, const Tensor& v_pages,
              const Tensor& table, const Tensor& q_start, const Tensor& kv_len) const {
    const int64_t rows = k0.dim() == 3 ? k0.size(0) : 0;
    for (int i = 0; i < 2; ++i) {
      const Tensor& t = i ? v0 : k0;
      check(i ? "v" : "k", t, 3, type, device);
      check_shape(i ? "v" : "k", t, {rows, args.heads_kv, args.head_dim});
    }
    const Tensor k = readable(k0), v = readable(v0);
    gpo_paged_args a = fill(rows, k_pages, v_pages, table, q_start, kv_len);
    a.k_new = heads3(k);
    a.v_new = heads3(v);
    launch("gpo_cache_append", gpo_cache_append, a, device);
  }

  Tensor attend(const Tensor& q0, const Tensor& k_pages, const Tensor& v_pages,
                const Tensor& table, const Tensor& q_start, const Tensor& kv_len,
                c10::optional<Tensor> out0, c10::optional<Tensor> lse) const {
    check("q", q0, 3, type, device);
    check_shape("q", q0, {q0.size(0), args.heads_q, args.head_dim});
    const Tensor q = readable(q0);
    if (out0) check_written("out", *out0, q.sizes(), type, device);
    if (lse) check_written("lse", *lse, q.sizes().slice(0, 2), at::kFloat, device);
    Tensor out = out0 ? *out0 : at::empty(q.sizes(), q.options());
    gpo_paged_args a = fill(q.size(0), k_pages, v_pages, table, q_start, kv_len);
    a.q = heads3(q);
    a.out = heads3(out);
    a.lse = lse ? static_cast<float*>(lse->data_ptr()) : nullptr;
    hold_workspace();
    launch("gpo_paged_attention", gpo_paged_attention, a, device);
    return out;
  }
};

}  // namespace

PYBIND11_MODULE(_ops, m) {
  m.def("set_refused", [](py::object cls) { g_refused = std::move(cls); });
  m.attr("ABI_VERSION") = GPO_ABI_VERSION;  // whose records this binding fills
  m.def("window_forward", &window_forward);
  m.def("window_backward", &window_backward);
  py::class_<Plan>(m, "Plan")
      .def(py::init([](int64_t hq, int64_t hk, int64_t d, int64_t page, int64_t seqs, int64_t max_q,
                       py::object dtype, c10::optional<int64_t> window, int64_t sinks,
                       c10::optional<double> scale, py::object device) {
        return std::make_unique<Plan>(hq, hk, d, page, seqs, max_q,
                                      torch::python::detail::py_object_to_dtype(dtype), window,
                                      sinks, scale,
                                      torch::python::detail::py_object_to_device(device));
      }))
      .def("append", &Plan::append)
      .def("attend", &Plan::attend);
  // the class outlives the interpreter's teardown order otherwise
  auto atexit = py::module_::import("atexit");
  atexit.attr("register")(py::cpp_function([] { g_refused = py::object(); }));
}
