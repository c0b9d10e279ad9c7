// PyTorch binding of the paged cache entries of include/fav4_bshd.h: the module behind fav4_bshd.paged.
//
// A decode step calls these a few times per layer on work that takes the GPU a few microseconds, so the
// host's share is kept small: arguments are read and checked here rather than in Python (a call costs the
// host about 4 us, of which the launch is half, against 25 us through ctypes).
//
// Workspaces: one for each device and stream, allocated from torch, its counters zeroed once, and kept; a
// call that is being captured into a CUDA graph gets one of the graph's own memory with a captured zeroing,
// so that replays on any stream disturb nobody.
#include <Python.h>
#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <cuda_runtime_api.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <climits>
#include <cmath>
#include <cstdint>
#include <initializer_list>
#include <map>
#include <utility>

#include "fav4_bshd.h"

namespace {

constexpr int64_t kHeadDim = 128;
constexpr int64_t kCounterBytes = 4096;

const at::Tensor& tensor_arg(PyObject* o, const char* name) {
  TORCH_CHECK_TYPE(THPVariable_Check(o), name, " must be a tensor, got ", Py_TYPE(o)->tp_name);
  return THPVariable_Unpack(o);
}
int64_t int_arg(PyObject* o, const char* name) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw python_error();
  TORCH_CHECK_VALUE(v >= INT_MIN && v <= INT_MAX, name, " is out of range: ", v);
  return v;
}
bool bool_arg(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw python_error();
  return v != 0;
}

int fits(int64_t v, const char* what) {
  TORCH_CHECK(v <= INT_MAX, what, " is out of range: ", v);
  return static_cast<int>(v);
}
const int* ints(const at::Tensor& t, const char* name, const at::Device& dev) {
  TORCH_CHECK(t.scalar_type() == at::kInt && t.device() == dev, name, " must be int32 on ", dev, ", got ",
              t.scalar_type(), " on ", t.device());
  return t.const_data_ptr<int>();
}
const int* row_ints(const at::Tensor& t, int64_t n, const char* name, const at::Device& dev) {
  TORCH_CHECK(t.dim() == 1 && t.size(0) == n && (n == 1 || t.stride(0) == 1), name, " must be [", n, "], contiguous, got ",
              t.sizes());
  return ints(t, name, dev);
}
// BF16 rows [T, heads, 128] with contiguous elements; the stride of a single entry says nothing
const void* rows(const at::Tensor& t, const char* name, const at::Device& dev, int64_t tokens, int64_t heads,
                 long long* token_stride, long long* head_stride) {
  TORCH_CHECK(t.dim() == 3 && t.size(2) == kHeadDim && (tokens < 0 || (t.size(0) == tokens && t.size(1) == heads)),
              name, " must be [T, heads, 128], got ", t.sizes());
  TORCH_CHECK(t.scalar_type() == at::kBFloat16 && t.device() == dev && t.stride(2) == 1, name,
              " must be bfloat16 on ", dev, " with contiguous elements");
  *token_stride = t.size(0) > 1 ? t.stride(0) : 0;
  *head_stride = t.size(1) > 1 ? t.stride(1) : 0;
  return t.const_data_ptr();
}
void no_grad(const char* what, std::initializer_list<const at::Tensor*> tensors) {
  if (at::GradMode::is_enabled())
    for (const at::Tensor* t : tensors)
      TORCH_CHECK(!t->requires_grad(), what, " has no gradient: call it under torch.no_grad(), or detach its inputs");
  if (c10::AutogradState::get_tls_state().get_fw_grad_mode())  // torch.no_grad() leaves forward mode on
    for (const at::Tensor* t : tensors)
      TORCH_CHECK(!t->_fw_grad(0).defined(), what, " has no gradient, forward-mode neither: unpack its dual inputs");
}
// A tensor that was written: an expression that saved it for its backward has to notice.
void written(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
// Whether two tensors of one shape lie in memory alike; the stride of a single entry says nothing.
bool same_layout(const at::Tensor& a, const at::Tensor& b) {
  for (int64_t d = 0; d < a.dim(); ++d)
    if (a.size(d) > 1 && a.stride(d) != b.stride(d)) return false;
  return true;
}
// Whether a contiguous result and an input share memory: other blocks still read rows where one writes its own.
bool overlap(const at::Tensor& out, const at::Tensor& in) {
  if (out.numel() == 0 || in.numel() == 0) return false;
  int64_t last = 0;
  for (int64_t d = 0; d < in.dim(); ++d) last += (in.size(d) - 1) * in.stride(d);
  const auto o = reinterpret_cast<uintptr_t>(out.const_data_ptr()), i = reinterpret_cast<uintptr_t>(in.const_data_ptr());
  return o < i + (last + 1) * in.element_size() && i < o + out.numel() * out.element_size();
}

Fav4PagedCache cache_of(PyObject* const* a, const at::Device& dev) {
  const at::Tensor& k = tensor_arg(a[0], "k_cache");
  const at::Tensor& v = tensor_arg(a[1], "v_cache");
  const at::Tensor& table = tensor_arg(a[2], "page_table");
  const at::Tensor& lens = tensor_arg(a[3], "seq_lens");
  TORCH_CHECK(k.dim() == 4 && k.size(3) == kHeadDim && v.sizes() == k.sizes() && same_layout(k, v),
              "k_cache and v_cache must be [pages, page_size, kv_heads, 128] of one layout, got ", k.sizes(), " and ",
              v.sizes());
  TORCH_CHECK(k.scalar_type() == at::kBFloat16 && v.scalar_type() == at::kBFloat16 && k.device() == dev &&
                  v.device() == dev && k.stride(3) == 1,
              "the caches must be bfloat16 on ", dev, " with contiguous elements");
  TORCH_CHECK(table.dim() == 2 && (table.size(1) <= 1 || table.stride(1) == 1),
              "page_table must be [B, max_pages] with contiguous rows, got ", table.sizes());
  Fav4PagedCache c;
  c.k = k.data_ptr();
  c.v = v.data_ptr();
  c.page_table = ints(table, "page_table", dev);
  c.seq_lens = row_ints(lens, table.size(0), "seq_lens", dev);
  c.page_stride = k.size(0) > 1 ? k.stride(0) : 0;
  c.token_stride = k.stride(1);
  c.head_stride = k.size(2) > 1 ? k.stride(2) : 0;
  c.table_stride = table.stride(0);
  c.batch = fits(table.size(0), "the batch");
  c.kv_heads = fits(k.size(2), "kv_heads");
  c.num_pages = fits(k.size(0), "the number of pages");
  c.page_size = fits(k.size(1), "page_size");
  c.max_pages = fits(table.size(1), "max_pages");
  return c;
}

void check_status(int status, const char* what) {
  TORCH_CHECK(status != 1, what, ": invalid arguments (CUDA status 1)");
  TORCH_CHECK(status == 0, what, ": CUDA status ", status);
}

at::Tensor workspace_for(size_t bytes, const at::Device& dev, cudaStream_t stream) {
  static auto* held = new std::map<std::pair<int, cudaStream_t>, at::Tensor>();  // kept to the end: CUDA may go first
  cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
  const cudaError_t e = cudaStreamIsCapturing(stream, &capture);
  TORCH_CHECK(e == cudaSuccess, "cudaStreamIsCapturing: ", cudaGetErrorString(e));
  const bool captured = capture != cudaStreamCaptureStatusNone;
  at::Tensor* kept = captured ? nullptr : &(*held)[{dev.index(), stream}];
  if (kept && kept->defined() && static_cast<size_t>(kept->numel()) >= bytes) return *kept;
  at::Tensor ws = at::empty({static_cast<int64_t>(bytes)}, at::TensorOptions().dtype(at::kByte).device(dev));
  ws.narrow(0, 0, kCounterBytes).zero_();
  if (kept) *kept = ws;
  return ws;
}

// append(q, k, v, k_cache, v_cache, page_table, seq_lens, cu_q, cos, sin, interleaved, offsets, out) -> Tensor
PyObject* append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 13, "append takes 13 arguments, got ", n);
  const at::Tensor& q = tensor_arg(a[0], "q");
  const at::Tensor& k = tensor_arg(a[1], "k");
  const at::Tensor& v = tensor_arg(a[2], "v");
  const at::Device dev = q.device();
  TORCH_CHECK(dev.is_cuda(), "q must be on a CUDA device, got ", dev);
  no_grad("append", {&q, &k, &v, &tensor_arg(a[3], "k_cache"), &tensor_arg(a[4], "v_cache")});
  const c10::cuda::CUDAGuard guard(dev);
  Fav4PagedAppendArgs p = {};
  p.cache = cache_of(a + 3, dev);
  p.q = rows(q, "q", dev, -1, 0, &p.q_token_stride, &p.q_head_stride);
  const int64_t tokens = q.size(0), heads = q.size(1);
  p.k = rows(k, "k", dev, tokens, p.cache.kv_heads, &p.k_token_stride, &p.k_head_stride);
  p.v = rows(v, "v", dev, tokens, p.cache.kv_heads, &p.v_token_stride, &p.v_head_stride);
  p.cu_seqlens_q = row_ints(tensor_arg(a[7], "cu_q"), static_cast<int64_t>(p.cache.batch) + 1, "cu_q", dev);
  TORCH_CHECK((a[8] == Py_None) == (a[9] == Py_None), "cos and sin come together");
  if (a[8] != Py_None) {
    const at::Tensor& c = tensor_arg(a[8], "cos");
    const at::Tensor& s = tensor_arg(a[9], "sin");
    no_grad("append", {&c, &s});
    TORCH_CHECK(c.dim() == 2 && s.sizes() == c.sizes() && c.is_contiguous() && s.is_contiguous() &&
                    c.scalar_type() == at::kFloat && s.scalar_type() == at::kFloat && c.device() == dev &&
                    s.device() == dev && c.size(1) >= 8 && c.size(1) % 8 == 0 && c.size(1) <= kHeadDim / 2,
                "cos and sin must be FP32 [positions, rotary / 2], contiguous, on ", dev,
                ", rotary a multiple of 16 up to 128; got ", c.sizes(), " and ", s.sizes());
    p.cos_table = c.const_data_ptr<float>();
    p.sin_table = s.const_data_ptr<float>();
    p.rotary_dim = static_cast<int>(2 * c.size(1));
    p.table_rows = fits(c.size(0), "the table");
  }
  p.interleaved = bool_arg(a[10]) ? 1 : 0;
  if (a[11] != Py_None) p.offsets = row_ints(tensor_arg(a[11], "offsets"), p.cache.batch, "offsets", dev);
  at::Tensor out;
  if (a[12] == Py_None) {
    out = at::empty({tokens, heads, kHeadDim}, q.options().requires_grad(false));
  } else {
    out = tensor_arg(a[12], "out");
    TORCH_CHECK(out.sizes() == q.sizes() && out.scalar_type() == at::kBFloat16 && out.device() == dev && out.is_contiguous(),
                "out must be contiguous bfloat16 of q's shape");
    no_grad("append", {&out});
    // a row of q may be turned in its own place
    TORCH_CHECK((q.is_contiguous() && out.const_data_ptr() == q.const_data_ptr()) || !overlap(out, q),
                "out may be q's own memory, but not a part of it");
    TORCH_CHECK(!overlap(out, k) && !overlap(out, v), "out must not overlap k or v");
    TORCH_CHECK(!overlap(out, tensor_arg(a[3], "k_cache")) && !overlap(out, tensor_arg(a[4], "v_cache")),
                "out must not overlap the caches");
  }
  p.q_out = out.data_ptr();
  p.heads = fits(heads, "heads");
  p.total_q = fits(tokens, "the number of tokens");
  check_status(fav4_bshd_paged_append(&p, c10::cuda::getCurrentCUDAStream(dev.index())), "paged append");
  written(tensor_arg(a[3], "k_cache"));
  written(tensor_arg(a[4], "v_cache"));
  if (a[12] != Py_None) written(out);
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// attend(q, k_cache, v_cache, page_table, seq_lens, cu_q, max_sq, causal, scale, out, return_lse, prefix_pages,
//        prefix_len) -> Tensor, or (Tensor, Tensor)
PyObject* attend(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 13, "attend takes 13 arguments, got ", n);
  const at::Tensor& q = tensor_arg(a[0], "q");
  const at::Device dev = q.device();
  TORCH_CHECK(dev.is_cuda(), "q must be on a CUDA device, got ", dev);
  no_grad("paged attention", {&q, &tensor_arg(a[1], "k_cache"), &tensor_arg(a[2], "v_cache")});
  const c10::cuda::CUDAGuard guard(dev);
  Fav4PagedArgs p = {};
  p.cache = cache_of(a + 1, dev);
  p.q = rows(q, "q", dev, -1, 0, &p.q_token_stride, &p.q_head_stride);
  const int64_t tokens = q.size(0), heads = q.size(1);
  p.cu_seqlens_q = row_ints(tensor_arg(a[5], "cu_q"), static_cast<int64_t>(p.cache.batch) + 1, "cu_q", dev);
  p.heads = fits(heads, "heads");
  p.total_q = fits(tokens, "the number of tokens");
  const int64_t max_sq = int_arg(a[6], "max_sq");
  TORCH_CHECK_VALUE(max_sq >= 0, "max_sq must not be negative, got ", max_sq);
  p.max_sq = static_cast<int>(max_sq < tokens ? max_sq : tokens);
  const bool causal = bool_arg(a[7]);
  if (a[8] == Py_None) {
    p.scale = 0.08838834764831845f;  // 1 / sqrt(128)
  } else {
    const double s = PyFloat_AsDouble(a[8]);
    if (s == -1.0 && PyErr_Occurred()) throw python_error();
    p.scale = static_cast<float>(s);
  }
  const bool prefixed = a[11] != Py_None;
  TORCH_CHECK(prefixed == (a[12] != Py_None), "prefix_pages and prefix_len come together");
  if (prefixed) {
    const at::Tensor& pages = tensor_arg(a[11], "prefix_pages");
    TORCH_CHECK(pages.dim() == 1, "prefix_pages must be [n], got ", pages.sizes());
    p.prefix_pages = row_ints(pages, pages.size(0), "prefix_pages", dev);
    p.max_prefix_pages = fits(pages.size(0), "prefix_pages");
    const at::Tensor& len = tensor_arg(a[12], "prefix_len");
    TORCH_CHECK(len.numel() == 1, "prefix_len must have one element, got ", len.sizes());
    p.prefix_len = ints(len, "prefix_len", dev);
  }
  at::Tensor out, lse;
  if (a[9] == Py_None) {
    out = at::empty({tokens, heads, kHeadDim}, q.options().requires_grad(false));
  } else {
    out = tensor_arg(a[9], "out");
    TORCH_CHECK(out.sizes() == q.sizes() && out.scalar_type() == at::kBFloat16 && out.device() == dev && out.is_contiguous(),
                "out must be contiguous bfloat16 of q's shape");
    no_grad("paged attention", {&out});
    TORCH_CHECK(!overlap(out, q), "out must not overlap q");
    TORCH_CHECK(!overlap(out, tensor_arg(a[1], "k_cache")) && !overlap(out, tensor_arg(a[2], "v_cache")),
                "out must not overlap the caches");
  }
  p.o = out.data_ptr();
  const bool with_lse = bool_arg(a[10]);
  if (with_lse) {
    lse = at::empty({heads, tokens}, q.options().dtype(at::kFloat).requires_grad(false));
    p.lse = lse.data_ptr<float>();
  }
  const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(dev.index());
  const size_t bytes = fav4_bshd_paged_workspace_bytes(&p);
  TORCH_CHECK(bytes > 0, "paged attention: invalid arguments");
  if (tokens > 0) {
    const at::Tensor ws = workspace_for(bytes, dev, stream);
    check_status((prefixed ? fav4_bshd_forward_shared_prefix : fav4_bshd_forward_paged)(&p, causal ? 1 : 0, ws.data_ptr(),
                                                                                      ws.numel(), stream),
                 "paged attention");
  }
  if (a[9] != Py_None) written(out);
  if (!with_lse) return THPVariable_Wrap(out);
  PyObject* both = PyTuple_New(2);
  if (!both) throw python_error();
  PyTuple_SET_ITEM(both, 0, THPVariable_Wrap(out));
  PyTuple_SET_ITEM(both, 1, THPVariable_Wrap(lse));
  return both;
  END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {
    {"append", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(append)), METH_FASTCALL, "fav4_bshd_paged_append"},
    {"attend", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(attend)), METH_FASTCALL,
     "fav4_bshd_forward_paged / fav4_bshd_forward_shared_prefix"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "fav4_paged_torch", "PyTorch binding of the paged cache", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_fav4_paged_torch() { return PyModule_Create(&module); }
