// Python binding of the paged 8-bit cache's three entry points for the calls that a server makes for every token and layer.
// A call of this module takes 4 us on the host for an append, 6 to 7 for a plan and 8 for a decode, where the same checks,
// tensors and ctypes structure take 20 to 33 us in Python; with kernels of 3 to 10 us that is what a decode step costs.
//
// Each function looks at its arguments and either launches and returns the result, or returns None without having done
// anything. None means "not this way": tensors that break a contract (Python then finds and names it), that need a copy
// first, that are traced or not ordinary tensors. Nothing here words an error but the library's own.
#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/GradMode.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/pybind.h>

#include <cmath>
#include <initializer_list>
#include <optional>
#include <stdexcept>
#include <string>

#include "../../include/fa_b200.h"

namespace py = pybind11;

namespace {

decltype(&fa_paged_plan) g_plan;
decltype(&fa_paged8_append) g_append;
decltype(&fa_decode_paged8) g_decode;
decltype(&fa_workspace_bytes) g_workspace;
decltype(&fa_last_error_string) g_error;

void bind(uint64_t plan, uint64_t append, uint64_t decode, uint64_t workspace, uint64_t error) {
  g_plan = reinterpret_cast<decltype(g_plan)>(plan);
  g_append = reinterpret_cast<decltype(g_append)>(append);
  g_decode = reinterpret_cast<decltype(g_decode)>(decode);
  g_workspace = reinterpret_cast<decltype(g_workspace)>(workspace);
  g_error = reinterpret_cast<decltype(g_error)>(error);
}

// The status words that Python made, by device.
constexpr int kMaxDevices = 64;
int32_t* g_status[kMaxDevices];
void set_status(int device, uint64_t word) {
  if (device >= 0 && device < kMaxDevices) g_status[device] = reinterpret_cast<int32_t*>(word);
}

// An ordinary CUDA tensor of `dims` dimensions (and `type`) on `device` (-1: any), or nullptr.
const at::Tensor* plain(py::handle h, int64_t dims, int device) {
  if (!THPVariable_CheckExact(h.ptr())) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(h.ptr());
  if (!t.is_cuda() || t.layout() != at::kStrided || t.dim() != dims) return nullptr;
  if (device >= 0 && t.get_device() != device) return nullptr;
  return &t;
}
const at::Tensor* plain(py::handle h, at::ScalarType type, int64_t dims, int device) {
  const at::Tensor* t = plain(h, dims, device);
  return t != nullptr && t->scalar_type() == type ? t : nullptr;
}

bool traced() { return c10::impl::TorchDispatchModeTLS::any_modes_set(); }
bool power_of_two(int64_t x) { return x > 0 && (x & (x - 1)) == 0; }

template <int N>
void strides_of(const at::Tensor& t, int64_t (&to)[N]) {
  for (int i = 0; i < N; ++i) to[i] = t.stride(i);
}

// (a, b, dim) 16-bit rows that the kernels read with 16-byte loads
bool rows16(const at::Tensor& t) {
  return t.stride(2) == 1 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 &&
         (t.size(0) <= 1 || t.stride(0) % 8 == 0) && (t.size(1) <= 1 || t.stride(1) % 8 == 0);
}

int dtype_of(const at::Tensor& t) {
  return t.scalar_type() == at::kHalf ? FA_F16 : t.scalar_type() == at::kBFloat16 ? FA_BF16 : -1;
}

bool needs_grad(std::initializer_list<const at::Tensor*> tensors) {
  if (!c10::GradMode::is_enabled()) return false;
  for (const at::Tensor* t : tensors)
    if (t->requires_grad()) return true;
  return false;
}

struct Cache {
  const at::Tensor *k, *v, *ks, *vs;
  int dtype;
  bool take(py::handle kc, py::handle vc, py::handle k_scales, py::handle v_scales, int device) {
    k = plain(kc, 4, device);
    v = plain(vc, 4, device);
    ks = plain(k_scales, at::kFloat, 2, device);
    vs = plain(v_scales, at::kFloat, 2, device);
    if (!k || !v || !ks || !vs || k->scalar_type() != v->scalar_type() || k->sizes() != v->sizes()) return false;
    dtype = k->scalar_type() == at::kFloat8_e4m3fn ? FA_CACHE_E4M3 : k->scalar_type() == at::kChar ? FA_CACHE_INT8 : -1;
    if (dtype < 0) return false;
    const int64_t blocks = k->size(0), bs = k->size(1), heads = k->size(2), dim = k->size(3);
    if (blocks <= 0 || heads <= 0 || blocks > INT32_MAX || !power_of_two(bs) || !power_of_two(dim) || dim < 16 || dim > 256)
      return false;
    for (const at::Tensor* t : {k, v}) {
      if (t->stride(3) != 1 || reinterpret_cast<uintptr_t>(t->data_ptr()) % 16) return false;
      for (int i = 0; i < 3; ++i)
        if (t->size(i) > 1 && (t->stride(i) <= 0 || t->stride(i) % 16)) return false;
    }
    for (const at::Tensor* t : {ks, vs})
      if (t->size(0) != blocks || t->size(1) != heads) return false;
    return true;
  }
};

// The launch on torch's current stream of the tensors' device.
template <typename F, typename P>
void launch(F fn, const P& p, int device) {
  const c10::cuda::OptionalCUDAGuard guard(
      device == c10::cuda::current_device() ? std::nullopt : std::optional<c10::Device>(c10::Device(c10::kCUDA, device)));
  const int32_t rc = fn(&p, c10::cuda::getCurrentCUDAStream(device).stream());
  if (rc) {
    const std::string message = "fa_b200 error " + std::to_string(rc) + ": " + g_error();
    throw std::runtime_error(message);
  }
}

at::Tensor empty(at::IntArrayRef sizes, at::ScalarType type, int device) {
  return at::detail::empty_cuda(sizes, type, c10::Device(c10::kCUDA, device), std::nullopt);
}

// A plain Python int (a bool is none), or -1.
int64_t index_of(py::handle h) {
  if (!PyLong_CheckExact(h.ptr())) return -1;
  const long long x = PyLong_AsLongLong(h.ptr());
  if (x == -1 && PyErr_Occurred()) PyErr_Clear();
  return x;
}

py::object plan(py::handle context_lens, py::handle new_lens, py::handle block_table, py::handle free_blocks,
                py::handle free_count, py::handle num_tokens_arg, py::handle block_size_arg, bool inplace) {
  const int64_t num_tokens = index_of(num_tokens_arg), block_size = index_of(block_size_arg);
  const at::Tensor* lens = plain(context_lens, at::kInt, 1, -1);
  if (!lens || traced()) return py::none();
  const int device = lens->get_device();
  const at::Tensor* fresh = plain(new_lens, at::kInt, 1, device);
  const at::Tensor* table = plain(block_table, at::kInt, 2, device);
  const at::Tensor* stack = plain(free_blocks, at::kInt, 1, device);
  const at::Tensor* count = plain(free_count, at::kInt, 1, device);
  if (!fresh || !table || !stack || !count) return py::none();
  const int64_t batch = lens->size(0), width = table->size(1);
  if (batch <= 0 || batch > FA_PLAN_MAX_BATCH || fresh->size(0) != batch || table->size(0) != batch || width <= 0 ||
      stack->size(0) <= 0 || stack->size(0) > INT32_MAX || count->size(0) != 1 || num_tokens < 0 ||
      num_tokens > INT32_MAX || !power_of_two(block_size) || block_size > INT32_MAX || width * block_size > INT32_MAX)
    return py::none();
  if (table->stride(1) != 1 || (batch > 1 && table->stride(0) < width) || stack->stride(0) != 1 ||
      (inplace && batch > 1 && lens->stride(0) != 1))
    return py::none();
  at::Tensor slots = empty({num_tokens}, at::kLong, device), cu = empty({batch + 1}, at::kInt, device);
  at::Tensor lens_out = inplace ? *lens : empty({batch}, at::kInt, device);
  at::Tensor count_out = inplace ? *count : empty({1}, at::kInt, device);
  fa_paged_plan_params p = {};
  p.batch = (int32_t)batch;
  p.max_blocks = (int32_t)width;
  p.num_blocks = (int32_t)stack->size(0);
  p.block_size = (int32_t)block_size;
  p.num_tokens = num_tokens;
  p.context_lens = static_cast<const int32_t*>(lens->data_ptr());
  p.cl_stride = lens->stride(0);
  p.new_lens = static_cast<const int32_t*>(fresh->data_ptr());
  p.nl_stride = fresh->stride(0);
  p.block_table = static_cast<int32_t*>(table->data_ptr());
  p.bt_stride = table->stride(0);
  p.free_blocks = static_cast<int32_t*>(stack->data_ptr());
  p.free_count = static_cast<const int32_t*>(count->data_ptr());
  p.slot_mapping = static_cast<int64_t*>(slots.data_ptr());
  p.cu_seqlens = static_cast<int32_t*>(cu.data_ptr());
  p.context_lens_out = static_cast<int32_t*>(lens_out.data_ptr());
  p.free_count_out = static_cast<int32_t*>(count_out.data_ptr());
  launch(g_plan, p, device);
  if (inplace) return py::make_tuple(slots, cu, py::reinterpret_borrow<py::object>(context_lens),
                                     py::reinterpret_borrow<py::object>(free_count));
  return py::make_tuple(slots, cu, lens_out, count_out);
}

// True when the launch was made.
bool append(py::handle key, py::handle value, py::handle k_cache, py::handle v_cache, py::handle k_scales,
            py::handle v_scales, py::handle slot_mapping) {
  const at::Tensor* k = plain(key, 3, -1);
  if (!k || traced()) return false;
  const int device = k->get_device();
  if (device >= kMaxDevices || g_status[device] == nullptr) return false;
  const at::Tensor* v = plain(value, k->scalar_type(), 3, device);
  const at::Tensor* slots = plain(slot_mapping, at::kLong, 1, device);
  Cache c;
  if (!v || !slots || dtype_of(*k) < 0 || !c.take(k_cache, v_cache, k_scales, v_scales, device)) return false;
  if (k->sizes() != v->sizes() || k->size(1) != c.k->size(2) || k->size(2) != c.k->size(3) || slots->size(0) != k->size(0) ||
      k->size(0) == 0 || !rows16(*k) || !rows16(*v))
    return false;
  for (const at::Tensor* t : {c.ks, c.vs})
    for (int i = 0; i < 2; ++i)
      if (t->size(i) > 1 && t->stride(i) <= 0) return false;
  if (needs_grad({k, v, c.k, c.v, c.ks, c.vs})) return false;
  fa_paged8_append_params p = {};
  p.dtype = dtype_of(*k);
  p.cache_dtype = c.dtype;
  p.heads_kv = (int32_t)k->size(1);
  p.head_dim = (int32_t)k->size(2);
  p.num_blocks = (int32_t)c.k->size(0);
  p.block_size = (int32_t)c.k->size(1);
  p.num_tokens = k->size(0);
  p.key = k->data_ptr();
  strides_of(*k, p.key_strides);
  p.value = v->data_ptr();
  strides_of(*v, p.value_strides);
  p.k_cache = c.k->data_ptr();
  strides_of(*c.k, p.k_strides);
  p.v_cache = c.v->data_ptr();
  strides_of(*c.v, p.v_strides);
  p.k_scales = static_cast<float*>(c.ks->data_ptr());
  strides_of(*c.ks, p.ks_strides);
  p.v_scales = static_cast<float*>(c.vs->data_ptr());
  strides_of(*c.vs, p.vs_strides);
  p.slot_mapping = static_cast<const int64_t*>(slots->data_ptr());
  p.slot_stride = slots->stride(0);
  p.status = g_status[device];
  launch(g_append, p, device);
  return true;
}

py::object decode(py::handle query, py::handle k_cache, py::handle v_cache, py::handle k_scales, py::handle v_scales,
                  py::handle block_table, py::handle context_lens, py::handle softmax_scale) {
  const at::Tensor* q = plain(query, 3, -1);
  if (!q || traced()) return py::none();
  if (!softmax_scale.is_none() && !(PyFloat_CheckExact(softmax_scale.ptr()) && std::isfinite(PyFloat_AS_DOUBLE(softmax_scale.ptr()))))
    return py::none();
  const int device = q->get_device();
  if (device >= kMaxDevices || g_status[device] == nullptr) return py::none();
  const at::Tensor* table = plain(block_table, at::kInt, 2, device);
  const at::Tensor* lens = plain(context_lens, at::kInt, 1, device);
  Cache c;
  if (!table || !lens || dtype_of(*q) < 0 || !c.take(k_cache, v_cache, k_scales, v_scales, device)) return py::none();
  const int64_t batch = q->size(0), heads = q->size(1), dim = q->size(2);
  if (batch <= 0 || heads <= 0 || batch > INT32_MAX || heads > INT32_MAX || dim != c.k->size(3) ||
      heads % c.k->size(2) || table->size(0) != batch || lens->size(0) != batch || table->size(1) <= 0 ||
      table->size(1) > INT32_MAX || !rows16(*q))
    return py::none();
  if (needs_grad({q, c.k, c.v, c.ks, c.vs})) return py::none();
  fa_paged8_params p = {};
  p.dtype = dtype_of(*q);
  p.cache_dtype = c.dtype;
  p.batch = (int32_t)batch;
  p.heads_q = (int32_t)heads;
  p.heads_kv = (int32_t)c.k->size(2);
  p.head_dim = (int32_t)dim;
  p.num_blocks = (int32_t)c.k->size(0);
  p.block_size = (int32_t)c.k->size(1);
  p.max_blocks = (int32_t)table->size(1);
  p.q = q->data_ptr();
  strides_of(*q, p.q_strides);
  p.k_cache = c.k->data_ptr();
  strides_of(*c.k, p.k_strides);
  p.v_cache = c.v->data_ptr();
  strides_of(*c.v, p.v_strides);
  p.k_scales = static_cast<const float*>(c.ks->data_ptr());
  strides_of(*c.ks, p.ks_strides);
  p.v_scales = static_cast<const float*>(c.vs->data_ptr());
  strides_of(*c.vs, p.vs_strides);
  p.block_table = static_cast<const int32_t*>(table->data_ptr());
  strides_of(*table, p.bt_strides);
  p.context_lens = static_cast<const int32_t*>(lens->data_ptr());
  p.cl_stride = lens->stride(0);
  p.softmax_scale = (float)(softmax_scale.is_none() ? 1.0 / std::sqrt((double)dim) : PyFloat_AS_DOUBLE(softmax_scale.ptr()));
  const c10::cuda::OptionalCUDAGuard guard(
      device == c10::cuda::current_device() ? std::nullopt : std::optional<c10::Device>(c10::Device(c10::kCUDA, device)));
  const int64_t bytes = g_workspace(FA_WS_PAGED8, &p);
  if (bytes < 0) return py::none();
  at::Tensor out = empty({batch, heads, dim}, q->scalar_type(), device), workspace = empty({bytes}, at::kByte, device);
  p.out = out.data_ptr();
  strides_of(out, p.o_strides);
  p.workspace = workspace.data_ptr();
  p.workspace_bytes = bytes;
  p.status = g_status[device];
  launch(g_decode, p, device);
  return py::cast(out);
}

}  // namespace

PYBIND11_MODULE(_paged_native, m) {
  m.attr("torch_version") = FA_TORCH;  // its headers are compiled in
  m.def("bind", &bind);
  m.def("set_status", &set_status);
  m.def("plan", &plan);
  m.def("append", &append);
  m.def("decode", &decode);
}
