// Python entry of the calls whose kernels are shorter than a Python argument check: the block-scaled
// cache, paged attention, page, norm and rotary operators.  Each function takes its arguments by position (the Python modules
// under ops/ name and document them), checks them, fills the C descriptor and calls the library's entry
// point on the current stream.  Nothing about a tensor is remembered between calls.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <array>
#include <cmath>
#include <cstdlib>
#include <cstring>
#include <initializer_list>
#include <map>
#include <memory>
#include <mutex>
#include <string>
#include <tuple>
#include <vector>

#include "mak_kvcache.h"

namespace {

// ---- the library's entry points, bound by address (the library itself is loaded by the package) --------
struct Library {
  decltype(&mak_last_error) last_error = nullptr;
  decltype(&mak_block_attention_workspace_bytes) workspace_bytes = nullptr;
  decltype(&mak_block_attention) attention = nullptr;
  decltype(&mak_block_append) append = nullptr;
  decltype(&mak_pages_fork) fork = nullptr;
  decltype(&mak_pages_grow) grow = nullptr;
  decltype(&mak_pages_free) free = nullptr;
  decltype(&mak_pages_compact) compact = nullptr;
  decltype(&mak_pages_copy) copy = nullptr;
  decltype(&mak_rope_axes) rope = nullptr;
  decltype(&mak_paged_attention_workspace_bytes) paged_workspace_bytes = nullptr;
  decltype(&mak_paged_attention) paged_attention = nullptr;
  decltype(&mak_paged_weights) paged_weights = nullptr;
  decltype(&mak_pages_evict) evict = nullptr;
  decltype(&mak_qk_norm_rope_partial_floats) norm_partial = nullptr;
  decltype(&mak_qk_norm_rope) norm_rope = nullptr;
} lib;
PyObject* emit = nullptr;  // dispatch.emit_native

using Args = PyObject* const*;

// A refusal: becomes ValueError, RuntimeError where `runtime`.
struct Refused {
  std::string text;
  bool runtime;
};
inline std::string text_of(const char* s) { return s; }
inline std::string text_of(const std::string& s) { return s; }
inline std::string text_of(int64_t v) { return std::to_string(v); }
inline std::string text_of(int v) { return std::to_string(v); }
template <typename... T>
std::string cat(const T&... parts) {
  return (std::string() + ... + text_of(parts));
}
template <typename... T>
[[noreturn]] void refuse(const char* name, const T&... parts) {
  throw Refused{cat(name, ": ", parts...), false};
}

const at::Tensor& tensor(const char* name, const char* what, PyObject* o) {
  if (!THPVariable_Check(o)) throw Refused{cat(name, ": ", what, " must be a tensor"), false};
  return THPVariable_Unpack(o);
}
int64_t integer(const char* name, const char* what, PyObject* o) {
  const int64_t v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    refuse(name, what, " must be an integer");
  }
  return v;
}
bool truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw python_error();
  return v == 1;
}
void count(const char* name, Py_ssize_t got, Py_ssize_t want) {
  if (got != want) throw Refused{cat(name, ": ", want, " arguments, got ", got), false};
}

// All on one CUDA device.
struct Device {
  const char* name;
  int index = -1;
  void add(const at::Tensor& t) {
    if (!t.is_cuda())
      throw Refused{cat(name, ": the B200 kvcache backend runs on CUDA tensors only (got a ", t.device().str(),
                        " tensor); there is no CPU fallback"), true};
    const int d = t.get_device();
    if (index < 0) index = d;
    if (d != index) refuse(name, "all tensors must be on the same device");
  }
  void need_library() const {
    if (lib.attention == nullptr) throw Refused{cat(name, ": musa_aiter kvcache native library missing"), true};
  }
};

void check(int rc, const char* name) {
  if (rc != 0) throw Refused{cat(name, ": native kernel library returned ", rc, ": ", lib.last_error()), true};
}

void trace(const char* op, PyObject* x, const char* reason) {
  const char* on = std::getenv("MUSA_AITER_TRACE_DISPATCH");
  if (on == nullptr || emit == nullptr) return;
  PyObject* r = PyObject_CallFunction(emit, "sOs", op, x, reason);
  if (r == nullptr) throw python_error();
  Py_DECREF(r);
}

// Runs f, turns what it throws into a Python exception.
template <typename F>
PyObject* guarded(F f) {
  HANDLE_TH_ERRORS
  try {
    return f();
  } catch (const Refused& r) {
    PyErr_SetString(r.runtime ? PyExc_RuntimeError : PyExc_ValueError, r.text.c_str());
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

at::Tensor empty(at::IntArrayRef shape, at::ScalarType dtype, const at::Device& device) {
  return at::empty(shape, at::TensorOptions().dtype(dtype).device(device));
}
PyObject* wrap(const at::Tensor& t) { return THPVariable_Wrap(t); }
PyObject* wrap(const at::Tensor& a, const at::Tensor& b) {
  PyObject* pair = PyTuple_New(2);
  if (pair == nullptr) throw python_error();
  PyTuple_SET_ITEM(pair, 0, THPVariable_Wrap(a));
  PyTuple_SET_ITEM(pair, 1, THPVariable_Wrap(b));
  return pair;
}

int float_code(at::ScalarType t) {
  return t == at::kHalf ? MAK_DT_F16 : t == at::kBFloat16 ? MAK_DT_BF16 : t == at::kFloat ? MAK_DT_F32 : -1;
}
// [rows, heads, dim] with contiguous, 16-byte aligned rows, copied where it has none.
at::Tensor aligned_rows(const at::Tensor& x) {
  const int64_t per = 16 / x.element_size();
  const auto st = x.strides();
  if (st[2] == 1 && st[0] % per == 0 && st[1] % per == 0 && reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0) return x;
  return x.clone(at::MemoryFormat::Contiguous);  // contiguous() would keep the stride of an axis with one entry, whatever it is
}

// Forward-mode differentiation has no formula here: a tangent that a tensor carries would be lost in silence.
void no_tangent(const char* name, std::initializer_list<const at::Tensor*> tensors) {
  if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
  for (const at::Tensor* t : tensors)
    if (t->defined() && t->_fw_grad(0).defined()) refuse(name, "no forward-mode derivative, but a tensor carries a tangent");
}

// ---- block-scaled caches --------------------------------------------------------------------------------

// Arguments from `a`: key_cache, value_cache, key_scale, value_scale, block_tables, context_lens, cu_seqlens.
mak_block_cache_desc cache_desc(const char* name, Args a, int64_t rows, int64_t head_dim, Device& dev) {
  const at::Tensor &kc = tensor(name, "key_cache", a[0]), &vc = tensor(name, "value_cache", a[1]);
  const at::Tensor &ks = tensor(name, "key_scale", a[2]), &vs = tensor(name, "value_scale", a[3]);
  const at::Tensor &table = tensor(name, "block_tables", a[4]), &ctx = tensor(name, "context_lens", a[5]);
  if (kc.dim() != 4 || kc.sizes() != vc.sizes())
    refuse(name, "key_cache and value_cache must both be [num_blocks, num_heads, head_dim, block_size]");
  const int64_t nb = kc.size(0), nh = kc.size(1), hd = kc.size(2), bs = kc.size(3);
  const at::ScalarType kind = kc.scalar_type();
  if ((kind != at::kChar && kind != at::kFloat8_e4m3fn) || vc.scalar_type() != kind)
    refuse(name, "caches must both be int8 or both float8_e4m3fn");
  if (hd != 64 && hd != 128 && hd != 256) refuse(name, "head_dim must be one of (64, 128, 256), got ", hd);
  if (bs != 16 && bs != 32 && bs != 64 && bs != 128) refuse(name, "block_size must be one of (16, 32, 64, 128), got ", bs);
  if (head_dim != hd) refuse(name, "rows have head_dim ", head_dim, ", the cache ", hd);
  if (nh < 1) refuse(name, "a cache needs heads");
  const auto kst = kc.strides(), vst = vc.strides();
  if (kst[3] != 1 || kst[2] != bs || vst[3] != 1 || vst[2] != bs)
    refuse(name, "the head_dim and block_size axes of the caches must be contiguous");
  for (const at::Tensor* s : {&ks, &vs}) {
    if (s->dim() != 2 || s->size(0) != nb || s->size(1) != nh) refuse(name, "scales must be [num_blocks, num_heads]");
    if (s->scalar_type() != at::kFloat) refuse(name, "scales must be float32");
  }
  if (table.dim() != 2 || ctx.dim() != 1 || table.size(0) != ctx.size(0))
    refuse(name, "block_tables must be [num_seqs, max_blocks] and context_lens [num_seqs]");
  if (table.scalar_type() != at::kInt || ctx.scalar_type() != at::kInt) refuse(name, "block_tables and context_lens must be int32");
  const int64_t seqs = table.size(0), width = table.size(1);
  if (width > 1 && table.stride(1) != 1) refuse(name, "a block table's row must be contiguous");
  if (seqs > 1 && ctx.stride(0) != 1) refuse(name, "context_lens must be contiguous");
  mak_block_cache_desc d = {};
  if (a[6] == Py_None) {
    if (rows != seqs) refuse(name, "without cu_seqlens every sequence has one row: ", rows, " rows for ", seqs, " sequences");
  } else {
    const at::Tensor& cu = tensor(name, "cu_seqlens", a[6]);
    if (cu.dim() != 1 || cu.size(0) != seqs + 1 || cu.scalar_type() != at::kInt) refuse(name, "cu_seqlens must be int32 [num_seqs + 1]");
    if (!cu.is_contiguous()) refuse(name, "cu_seqlens must be contiguous");
    dev.add(cu);
    d.cu_seqlens = static_cast<const int32_t*>(cu.data_ptr());
  }
  for (const at::Tensor* t : {&kc, &vc, &ks, &vs, &table, &ctx}) dev.add(*t);
  d.key = kc.data_ptr(), d.value = vc.data_ptr();
  d.key_scale = static_cast<float*>(ks.data_ptr()), d.value_scale = static_cast<float*>(vs.data_ptr());
  // the stride of an axis with one entry reaches nothing: a multiple of 16 in its place
  auto step = [&](at::IntArrayRef st, int64_t axis, int64_t size) { return size > 1 ? st[axis] : nh * hd * bs; };
  d.key_stride_block = step(kst, 0, nb), d.key_stride_head = step(kst, 1, nh);
  d.value_stride_block = step(vst, 0, nb), d.value_stride_head = step(vst, 1, nh);
  d.key_scale_stride_block = ks.stride(0), d.key_scale_stride_head = ks.stride(1);
  d.value_scale_stride_block = vs.stride(0), d.value_scale_stride_head = vs.stride(1);
  d.block_tables = static_cast<const int32_t*>(table.data_ptr());
  d.context_lens = static_cast<const int32_t*>(ctx.data_ptr());
  d.table_stride = table.stride(0);
  d.num_blocks = nb, d.num_seqs = seqs, d.max_blocks = width, d.num_rows = rows;
  d.num_heads = static_cast<int32_t>(nh), d.head_dim = static_cast<int32_t>(hd), d.block_size = static_cast<int32_t>(bs);
  d.code_type = kind == at::kChar ? MAK_CODE_INT8 : MAK_CODE_E4M3;
  return d;
}

// Attention workspaces, one per device and stream: the kernels leave their counters at zero, so calls that
// follow one another on a stream share it.  The per-thread default stream is another one for each thread, under one
// handle.  Kept until the process ends.
struct Workspaces {
  std::mutex mutex;
  std::map<std::tuple<int, cudaStream_t, const void*>, at::Tensor> kept;
};
at::Tensor workspace(Workspaces& all, int64_t bytes, const at::Device& device, cudaStream_t stream) {
  static thread_local char thread;
  if (c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None) {
    // a graph may be replayed on any stream: it gets a workspace of its own
    at::Tensor ws = empty({bytes}, at::kByte, device);
    ws.narrow(0, 0, std::min<int64_t>(bytes, 1 << 16)).zero_();
    return ws;
  }
  std::lock_guard<std::mutex> lock(all.mutex);
  at::Tensor& ws = all.kept[{device.index(), stream, stream == cudaStreamPerThread ? &thread : nullptr}];
  if (!ws.defined()) ws = at::zeros({bytes}, at::TensorOptions().dtype(at::kByte).device(device));
  return ws;
}

// q, the seven of cache_desc, scale (None: 1 / sqrt(head_dim)), causal, window, return_lse, out (or None)
PyObject* py_attend(PyObject*, Args a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    const char* name = "paged_attention_block_scaled";
    count(name, n, 13);
    const at::Tensor& q0 = tensor(name, "q", a[0]);
    if (q0.dim() != 3) refuse(name, "q must be [rows, num_q_heads, head_dim]");
    const at::ScalarType kind = q0.scalar_type();
    if (kind != at::kHalf && kind != at::kBFloat16) refuse(name, "q must be float16 or bfloat16, got ", toString(kind));
    const int64_t rows = q0.size(0), hq = q0.size(1), hd = q0.size(2);
    const bool causal = truth(a[9]), want_lse = truth(a[11]);
    const int64_t window = integer(name, "window", a[10]);
    if (window < 0 || (window && !causal)) refuse(name, "window must be positive or 0 and needs causal=True");
    Device dev{name};
    mak_block_attn_desc d = {};
    const at::Tensor& kc = tensor(name, "key_cache", a[1]);
    if (kc.dim() == 4 && kc.size(1) > 0 && (hq < 1 || hq % kc.size(1)))
      refuse(name, hq, " query heads do not divide over ", kc.size(1), " cache heads");
    const bool given = a[12] != Py_None;
    if (given) {
      const at::Tensor& o = tensor(name, "out", a[12]);
      if (o.sizes() != q0.sizes() || o.scalar_type() != kind || (o.numel() && o.stride(2) != 1))
        refuse(name, "out must have q's shape and dtype and contiguous rows");
    }
    d.cache = cache_desc(name, a + 1, rows, hd, dev);
    dev.add(q0);
    if (given) dev.add(THPVariable_Unpack(a[12]));
    dev.need_library();
    const c10::cuda::CUDAGuard on(static_cast<c10::DeviceIndex>(dev.index));
    const at::Tensor q = aligned_rows(q0);
    const at::Tensor out = given ? THPVariable_Unpack(a[12]) : empty({rows, hq, hd}, kind, q0.device());
    const at::Tensor lse = want_lse ? empty({rows, hq}, at::kFloat, q0.device()) : at::Tensor();
    const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(dev.index)).stream();
    static auto* spaces = new Workspaces();
    const at::Tensor ws = workspace(*spaces, lib.workspace_bytes(), q0.device(), stream);
    d.q = q.data_ptr(), d.out = out.data_ptr(), d.lse = want_lse ? static_cast<float*>(lse.data_ptr()) : nullptr;
    d.workspace = ws.data_ptr(), d.workspace_bytes = ws.numel();
    d.q_stride_row = q.stride(0), d.q_stride_head = q.stride(1), d.out_stride_row = out.stride(0), d.out_stride_head = out.stride(1);
    d.num_q_heads = static_cast<int32_t>(hq), d.q_dtype = float_code(kind), d.causal = causal;
    d.window = static_cast<int32_t>(std::min<int64_t>(window, 0x7fffffff));
    double scale = 1.0 / std::sqrt(static_cast<double>(hd));
    if (a[8] != Py_None) {
      scale = PyFloat_AsDouble(a[8]);
      if (scale == -1.0 && PyErr_Occurred()) throw python_error();
    }
    d.scale = static_cast<float>(scale);
    check(lib.attention(&d, stream), name);
    trace(name, a[0], "sm100a block-scaled cache attention");
    return want_lse ? wrap(out, lse) : wrap(out);
  });
}

// k, v, the seven of cache_desc
PyObject* py_append(PyObject*, Args a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    const char* name = "kv_append_block_scaled";
    count(name, n, 9);
    const at::Tensor &k0 = tensor(name, "k", a[0]), &v0 = tensor(name, "v", a[1]);
    if (k0.dim() != 3 || k0.sizes() != v0.sizes()) refuse(name, "k and v must both be [rows, num_heads, head_dim]");
    const int code = float_code(k0.scalar_type());
    if (code < 0 || v0.scalar_type() != k0.scalar_type()) refuse(name, "k and v must both be float16, bfloat16 or float32");
    Device dev{name};
    const mak_block_cache_desc d = cache_desc(name, a + 2, k0.size(0), k0.size(2), dev);
    if (d.num_heads != k0.size(1)) refuse(name, "rows have ", k0.size(1), " heads, the cache ", d.num_heads);
    dev.add(k0);
    dev.add(v0);
    dev.need_library();
    const c10::cuda::CUDAGuard on(static_cast<c10::DeviceIndex>(dev.index));
    const at::Tensor k = aligned_rows(k0), v = aligned_rows(v0);
    check(lib.append(&d, k.data_ptr(), v.data_ptr(), k.stride(0), k.stride(1), v.stride(0), v.stride(1), code,
                     c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(dev.index)).stream()),
          name);
    trace(name, a[0], "sm100a block-scaled cache writer");
    Py_RETURN_NONE;
  });
}

// ---- pages ------------------------------------------------------------------------------------------------

int32_t* index_of(const char* name, const char* what, const at::Tensor& t, int64_t dim, Device& dev) {
  if (t.dim() != dim || t.scalar_type() != at::kInt)
    refuse(name, what, " must be an int32 tensor of ", dim, dim > 1 ? " dimensions" : " dimension");
  if (t.numel() > 1 && t.size(-1) > 1 && t.stride(-1) != 1) refuse(name, what, " must be contiguous");
  (void)dev;
  return static_cast<int32_t*>(t.data_ptr());
}

mak_pages_desc pool(const char* name, const at::Tensor& table, const at::Tensor* lens, const at::Tensor& refs, int64_t block_size,
                    Device& dev) {
  mak_pages_desc d = {};
  d.block_tables = index_of(name, "block_tables", table, 2, dev);
  d.ref_counts = index_of(name, "ref_counts", refs, 1, dev);
  if (lens != nullptr) {
    d.context_lens = index_of(name, "context_lens", *lens, 1, dev);
    if (lens->size(0) != table.size(0)) refuse(name, "context_lens must have one entry per row of block_tables");
  }
  if (block_size <= 0) refuse(name, "block_size must be positive");
  d.table_stride = table.stride(0), d.num_rows = table.size(0), d.max_blocks = table.size(1), d.num_pages = refs.size(0);
  d.block_size = block_size;
  return d;
}

// The tensors of a sequence of planes as mak_pages_planes.
struct Planes {
  std::vector<uint64_t> ptrs;
  std::vector<int64_t> strides, sizes;
  std::vector<const at::Tensor*> tensors;
  PyObject* held = nullptr;
  mak_pages_planes desc = {};
  Planes(const char* name, PyObject* sequence, int64_t pages) {
    held = PySequence_Fast(sequence, "planes must be a sequence of tensors");
    if (held == nullptr) throw python_error();
    const Py_ssize_t n = PySequence_Fast_GET_SIZE(held);
    ptrs.reserve(n), strides.reserve(n), sizes.reserve(n), tensors.reserve(n);
    try {
      for (Py_ssize_t i = 0; i < n; ++i) {
        const at::Tensor& t = tensor(name, "a plane", PySequence_Fast_GET_ITEM(held, i));
        if (t.dim() == 0 || t.size(0) != pages) refuse(name, "every plane's first axis must have ", pages, " pages");
        const int64_t per = pages ? t.numel() / pages : 0, item = t.element_size();
        int64_t step = per;
        if (!t.is_contiguous()) {
          int64_t want = 1;
          for (int64_t d = t.dim() - 1; d > 0; --d) {
            if (t.size(d) != 1 && t.stride(d) != want) refuse(name, "a page of a plane must be contiguous");
            want *= t.size(d);
          }
          if (t.stride(0) < per) refuse(name, "pages of a plane must not overlap");
          step = t.stride(0);
        }
        ptrs.push_back(reinterpret_cast<uintptr_t>(t.data_ptr()));
        strides.push_back(step * item);
        sizes.push_back(per * item);
        tensors.push_back(&t);
      }
    } catch (...) {
      Py_DECREF(held);
      throw;
    }
    desc = {ptrs.data(), strides.data(), sizes.data(), static_cast<int64_t>(n)};
  }
  Planes(const Planes&) = delete;
  Planes& operator=(const Planes&) = delete;
  ~Planes() { Py_DECREF(held); }
  void on(Device& dev) const {
    for (const at::Tensor* t : tensors) dev.add(*t);
  }
};

cudaStream_t stream_of(const Device& dev) {
  return c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(dev.index)).stream();
}

// block_tables, context_lens, parents, children, ref_counts, planes, block_size
PyObject* py_fork(PyObject*, Args a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    const char* name = "kv_pages_fork";
    count(name, n, 7);
    const at::Tensor &table = tensor(name, "block_tables", a[0]), &lens = tensor(name, "context_lens", a[1]);
    const at::Tensor &parents = tensor(name, "parents", a[2]), &children = tensor(name, "children", a[3]);
    const at::Tensor& refs = tensor(name, "ref_counts", a[4]);
    Device dev{name};
    const mak_pages_desc d = pool(name, table, &lens, refs, integer(name, "block_size", a[6]), dev);
    const int32_t *from = index_of(name, "parents", parents, 1, dev), *to = index_of(name, "children", children, 1, dev);
    const int64_t want = parents.size(0);
    if (children.size(0) != want) refuse(name, "parents and children must have the same length");
    const Planes planes(name, a[5], refs.size(0));
    for (const at::Tensor* t : {&table, &lens, &parents, &children, &refs}) dev.add(*t);
    planes.on(dev);
    dev.need_library();
    const c10::cuda::CUDAGuard on(static_cast<c10::DeviceIndex>(dev.index));
    // the answer and the scratch in one allocation
    const at::Tensor room = empty({2 * want + 4}, at::kInt, table.device());
    int32_t* at = static_cast<int32_t*>(room.data_ptr());
    check(lib.fork(&d, &planes.desc, from, to, want, at, at + 1, stream_of(dev)), name);
    trace(name, a[0], "sm100a page fork");
    return wrap(room.narrow(0, 0, 1));
  });
}

// block_tables, context_lens, rows, new_tokens, ref_counts, block_size
PyObject* py_grow(PyObject*, Args a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    const char* name = "kv_pages_grow";
    count(name, n, 6);
    const at::Tensor &table = tensor(name, "block_tables", a[0]), &lens = tensor(name, "context_lens", a[1]);
    const at::Tensor &rows = tensor(name, "rows", a[2]), &more = tensor(name, "new_tokens", a[3]);
    const at::Tensor& refs = tensor(name, "ref_counts", a[4]);
    Device dev{name};
    const mak_pages_desc d = pool(name, table, &lens, refs, integer(name, "block_size", a[5]), dev);
    const int32_t *r = index_of(name, "rows", rows, 1, dev), *m = index_of(name, "new_tokens", more, 1, dev);
    if (rows.size(0) != more.size(0)) refuse(name, "rows and new_tokens must have the same length");
    for (const at::Tensor* t : {&table, &lens, &rows, &more, &refs}) dev.add(*t);
    dev.need_library();
    const c10::cuda::CUDAGuard on(static_cast<c10::DeviceIndex>(dev.index));
    const at::Tensor missing = empty({1}, at::kInt, table.device());
    check(lib.grow(&d, r, m, rows.size(0), static_cast<int32_t*>(missing.data_ptr()), stream_of(dev)), name);
    trace(name, a[0], "sm100a page growth");
    return wrap(missing);
  });
}

// block_tables, context_lens, rows, ref_counts
PyObject* py_free(PyObject*, Args a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    const char* name = "kv_pages_free";
    count(name, n, 4);
    const at::Tensor &table = tensor(name, "block_tables", a[0]), &lens = tensor(name, "context_lens", a[1]);
    const at::Tensor &rows = tensor(name, "rows", a[2]), &refs = tensor(name, "ref_counts", a[3]);
    Device dev{name};
    const mak_pages_desc d = pool(name, table, &lens, refs, 1, dev);
    const int32_t* r = index_of(name, "rows", rows, 1, dev);
    for (const at::Tensor* t : {&table, &lens, &rows, &refs}) dev.add(*t);
    dev.need_library();
    const c10::cuda::CUDAGuard on(static_cast<c10::DeviceIndex>(dev.index));
    check(lib.free(&d, r, rows.size(0), stream_of(dev)), name);
    trace(name, a[0], "sm100a page release");
    Py_RETURN_NONE;
  });
}

// block_tables, ref_counts, planes
PyObject* py_compact(PyObject*, Args a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    const char* name = "kv_pages_compact";
    count(name, n, 3);
    const at::Tensor &table = tensor(name, "block_tables", a[0]), &refs = tensor(name, "ref_counts", a[1]);
    Device dev{name};
    const mak_pages_desc d = pool(name, table, nullptr, refs, 1, dev);
    const Planes planes(name, a[2], refs.size(0));
    dev.add(table);
    dev.add(refs);
    planes.on(dev);
    dev.need_library();
    const c10::cuda::CUDAGuard on(static_cast<c10::DeviceIndex>(dev.index));
    const at::Tensor live = empty({1}, at::kInt, table.device());
    const at::Tensor scratch = empty({3 * refs.size(0) + 2}, at::kInt, table.device());
    check(lib.compact(&d, &planes.desc, static_cast<int32_t*>(live.data_ptr()), static_cast<int32_t*>(scratch.data_ptr()), stream_of(dev)),
          name);
    trace(name, a[0], "sm100a page compaction");
    return wrap(live);
  });
}

// planes, src_pages, dst_pages
PyObject* py_copy(PyObject*, Args a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    const char* name = "kv_pages_copy";
    count(name, n, 3);
    const at::Tensor &src = tensor(name, "src_pages", a[1]), &dst = tensor(name, "dst_pages", a[2]);
    Device dev{name};
    const int32_t *s = index_of(name, "src_pages", src, 1, dev), *d = index_of(name, "dst_pages", dst, 1, dev);
    if (src.size(0) != dst.size(0)) refuse(name, "src_pages and dst_pages must have the same length");
    int64_t pages = 0;
    {
      PyObject* first = PySequence_Size(a[0]) > 0 ? PySequence_GetItem(a[0], 0) : nullptr;
      if (first != nullptr) {
        if (THPVariable_Check(first) && THPVariable_Unpack(first).dim() > 0) pages = THPVariable_Unpack(first).size(0);
        Py_DECREF(first);
      } else if (PyErr_Occurred()) {
        throw python_error();
      }
    }
    const Planes planes(name, a[0], pages);
    if (planes.tensors.empty()) Py_RETURN_NONE;
    dev.add(src);
    dev.add(dst);
    planes.on(dev);
    dev.need_library();
    const c10::cuda::CUDAGuard on(static_cast<c10::DeviceIndex>(dev.index));
    check(lib.copy(&planes.desc, pages, s, d, src.size(0), stream_of(dev)), name);
    trace(name, a[1], "sm100a page copy");
    Py_RETURN_NONE;
  });
}

// ---- rotary positions ---------------------------------------------------------------------------------------

// q, k, positions, cos, sin, sections, interleaved, interleaved_axes, inverse; None where q or k wants a gradient
PyObject* py_rope(PyObject*, Args a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    const bool inverse = n == 9 && truth(a[8]);
    const char* name = inverse ? "apply_rope_axes_backward" : "apply_rope_axes";
    count(name, n, 9);
    const at::Tensor &q0 = tensor(name, "q", a[0]), &k0 = tensor(name, "k", a[1]);
    at::Tensor pos = tensor(name, "positions", a[2]), cos = tensor(name, "cos", a[3]), sin = tensor(name, "sin", a[4]);
    no_tangent(name, {&q0, &k0, &cos, &sin});
    if (c10::GradMode::is_enabled()) {
      if (cos.requires_grad() || sin.requires_grad()) refuse(name, "cos and sin are tables without a gradient, detach them");
      if (q0.requires_grad() || k0.requires_grad()) Py_RETURN_NONE;  // the caller's autograd function calls again, with gradients off
    }
    if (q0.dim() != 3 || k0.dim() != 3 || q0.size(0) != k0.size(0) || q0.size(2) != k0.size(2))
      refuse(name, "q and k must be [tokens, heads, head_dim] with the same tokens and head_dim");
    const at::ScalarType kind = q0.scalar_type();
    if ((kind != at::kHalf && kind != at::kBFloat16) || k0.scalar_type() != kind)
      refuse(name, "q and k must both be float16 or both bfloat16");
    const int64_t tokens = q0.size(0), hq = q0.size(1), hk = k0.size(1), hd = q0.size(2);
    const bool inter = truth(a[6]), dealt = truth(a[7]);
    mak_rope_axes_desc d = {};
    // axis of each pair: the sections one after another, or dealt out in turn while one has pairs left
    std::vector<int64_t> sections;
    {
      PyObject* seq = PySequence_Fast(a[5], "sections must be a sequence");
      if (seq == nullptr) throw python_error();
      const Py_ssize_t axes = PySequence_Fast_GET_SIZE(seq);
      bool fine = axes > 0 && axes < 256;
      for (Py_ssize_t i = 0; fine && i < axes; ++i) {
        const int64_t s = PyLong_AsLongLong(PySequence_Fast_GET_ITEM(seq, i));
        if (s == -1 && PyErr_Occurred()) PyErr_Clear();
        fine = s >= 0;
        sections.push_back(s);
      }
      Py_DECREF(seq);
      if (!fine) refuse(name, "sections must be counts of pairs, one per axis");
    }
    int64_t half = 0;
    for (int64_t s : sections) half += std::min<int64_t>(s, 1 << 20);
    const int64_t unit = inter ? 4 : 8;
    if (half == 0 || 2 * half > hd || half > MAK_ROPE_MAX_PAIRS || half % unit || hd % 8)
      refuse(name, "sections must add up to a multiple of ", unit, " pairs, at most head_dim / 2 and ", MAK_ROPE_MAX_PAIRS, ", got ", half,
             " with head_dim ", hd, " (a multiple of 8)");
    if (!dealt) {
      int64_t at = 0;
      for (size_t x = 0; x < sections.size(); ++x)
        for (int64_t i = 0; i < sections[x]; ++i) d.pair_axis[at++] = static_cast<uint8_t>(x);
    } else {
      std::vector<int64_t> left = sections;
      for (int64_t at = 0; at < half;)
        for (size_t x = 0; x < left.size(); ++x)
          if (left[x] > 0) {
            --left[x];
            d.pair_axis[at++] = static_cast<uint8_t>(x);
          }
    }
    const int64_t axes = static_cast<int64_t>(sections.size());
    if (pos.dim() != 2 || pos.size(0) != axes || pos.size(1) != tokens || (pos.scalar_type() != at::kInt && pos.scalar_type() != at::kLong))
      refuse(name, "positions must be int32 or int64 [", axes, ", ", tokens, "]");
    if (cos.dim() != 2 || cos.sizes() != sin.sizes() || cos.size(1) != half) refuse(name, "cos and sin must both be [max_positions, ", half, "]");
    if (cos.scalar_type() != at::kFloat || sin.scalar_type() != at::kFloat) refuse(name, "cos and sin must be float32");
    Device dev{name};
    for (const at::Tensor* t : {&q0, &k0, static_cast<const at::Tensor*>(&pos), static_cast<const at::Tensor*>(&cos),
                                static_cast<const at::Tensor*>(&sin)})
      dev.add(*t);
    dev.need_library();
    const c10::cuda::CUDAGuard on(static_cast<c10::DeviceIndex>(dev.index));
    const at::Tensor q = aligned_rows(q0), k = aligned_rows(k0);
    if (tokens > 1 && pos.stride(1) != 1) pos = pos.contiguous();
    if (cos.stride(1) != 1) cos = cos.contiguous();
    if (sin.stride(1) != 1) sin = sin.contiguous();
    const at::Tensor q_out = empty({tokens, hq, hd}, kind, q0.device()), k_out = empty({tokens, hk, hd}, kind, q0.device());
    d.q = q.data_ptr(), d.k = hk ? k.data_ptr() : nullptr, d.q_out = q_out.data_ptr(), d.k_out = k_out.data_ptr();
    d.positions = pos.data_ptr(), d.cos = static_cast<const float*>(cos.data_ptr()), d.sin = static_cast<const float*>(sin.data_ptr());
    d.tokens = tokens, d.max_positions = cos.size(0);
    d.q_stride_token = q.stride(0), d.q_stride_head = q.stride(1), d.k_stride_token = k.stride(0), d.k_stride_head = k.stride(1);
    d.qo_stride_token = hq * hd, d.qo_stride_head = hd, d.ko_stride_token = hk * hd, d.ko_stride_head = hd;
    d.pos_stride = pos.stride(0), d.cos_stride = cos.stride(0), d.sin_stride = sin.stride(0);
    d.q_heads = static_cast<int32_t>(hq), d.k_heads = static_cast<int32_t>(hk), d.head_dim = static_cast<int32_t>(hd);
    d.rot_dim = static_cast<int32_t>(2 * half), d.dtype = float_code(kind);
    d.pos_dtype = pos.scalar_type() == at::kInt ? MAK_DT_I32 : MAK_DT_I64;
    d.axes = static_cast<int32_t>(axes), d.interleaved = inter, d.inverse = inverse;
    check(lib.rope(&d, stream_of(dev)), name);
    trace(name, a[0], "sm100a rotary positions with several axes");
    return wrap(q_out, k_out);
  });
}

// ---- paged 16-bit caches ----------------------------------------------------------------------------------

// Arguments from `a`: key_cache, value_cache (where `values`), block_tables, context_lens; `cu`: cu_seqlens.
// The tensors go to `used`: whether they are on one device is asked after all shapes.
using Used = std::vector<const at::Tensor*>;
mak_paged_cache_desc paged_desc(const char* name, Args a, bool values, PyObject* cu_seqlens, const at::Tensor& q, Used& used) {
  const at::Tensor& kc = tensor(name, "key_cache", a[0]);
  const at::Tensor& vc = values ? tensor(name, "value_cache", a[1]) : kc;
  a += values ? 2 : 1;
  const at::Tensor &table = tensor(name, "block_tables", a[0]), &ctx = tensor(name, "context_lens", a[1]);
  if (q.dim() != 3) refuse(name, "q must be [rows, num_q_heads, head_dim]");
  const at::ScalarType kind = q.scalar_type();
  if (kind != at::kHalf && kind != at::kBFloat16) refuse(name, "q must be float16 or bfloat16, got ", toString(kind));
  if (kc.dim() != 4 || kc.sizes() != vc.sizes())
    refuse(name, values ? "key_cache and value_cache must both be" : "key_cache must be", " [num_blocks, block_size, num_heads, head_dim]");
  if (kc.scalar_type() != kind || vc.scalar_type() != kind) refuse(name, "q and the caches must have one type, got ", toString(kind), " and ", toString(kc.scalar_type()));
  const int64_t rows = q.size(0), hq = q.size(1), nb = kc.size(0), bs = kc.size(1), nh = kc.size(2), hd = kc.size(3);
  if (hd != 64 && hd != 128) refuse(name, "head_dim must be one of (64, 128), got ", hd);
  if (bs != 16 && bs != 32 && bs != 64 && bs != 128) refuse(name, "block_size must be one of (16, 32, 64, 128), got ", bs);
  if (q.size(2) != hd) refuse(name, "rows have head_dim ", q.size(2), ", the cache ", hd);
  if (nh < 1) refuse(name, "a cache needs heads");
  if (hq < 1 || hq % nh) refuse(name, hq, " query heads do not divide over ", nh, " cache heads");
  for (const at::Tensor* c : {&kc, &vc}) {
    if (c->stride(3) != 1) refuse(name, "the head_dim axis of the caches must be contiguous");
    if (nb == 0) continue;
    for (int i = 0; i < 3; ++i)
      if (c->size(i) > 1 && c->stride(i) % 8) refuse(name, "block, token and head strides of the caches must be multiples of 8 elements");
    if (reinterpret_cast<uintptr_t>(c->data_ptr()) % 16) refuse(name, "caches must begin on 16 bytes");
  }
  if (table.dim() != 2 || ctx.dim() != 1 || table.size(0) != ctx.size(0))
    refuse(name, "block_tables must be [num_seqs, max_blocks] and context_lens [num_seqs]");
  if (table.scalar_type() != at::kInt || ctx.scalar_type() != at::kInt) refuse(name, "block_tables and context_lens must be int32");
  const int64_t seqs = table.size(0), width = table.size(1);
  if (width > 1 && table.stride(1) != 1) refuse(name, "a block table's row must be contiguous");
  if (seqs > 1 && ctx.stride(0) != 1) refuse(name, "context_lens must be contiguous");
  mak_paged_cache_desc d = {};
  if (cu_seqlens == Py_None) {
    if (rows != seqs) refuse(name, "without cu_seqlens every sequence has one row: ", rows, " rows for ", seqs, " sequences");
  } else {
    const at::Tensor& cu = tensor(name, "cu_seqlens", cu_seqlens);
    if (cu.dim() != 1 || cu.size(0) != seqs + 1 || cu.scalar_type() != at::kInt) refuse(name, "cu_seqlens must be int32 [num_seqs + 1]");
    if (!cu.is_contiguous()) refuse(name, "cu_seqlens must be contiguous");
    used.push_back(&cu);
    d.cu_seqlens = static_cast<const int32_t*>(cu.data_ptr());
  }
  for (const at::Tensor* t : {&kc, &vc, &table, &ctx, &q}) used.push_back(t);
  d.key = kc.data_ptr(), d.value = values ? vc.data_ptr() : nullptr;
  // the stride of an axis with one entry reaches nothing: a multiple of 8 in its place
  auto step = [&](const at::Tensor& c, int axis) { return c.size(axis) > 1 ? c.stride(axis) : nh * hd * bs; };
  d.key_stride_block = step(kc, 0), d.key_stride_token = step(kc, 1), d.key_stride_head = step(kc, 2);
  d.value_stride_block = step(vc, 0), d.value_stride_token = step(vc, 1), d.value_stride_head = step(vc, 2);
  d.block_tables = static_cast<const int32_t*>(table.data_ptr());
  d.context_lens = static_cast<const int32_t*>(ctx.data_ptr());
  d.table_stride = table.stride(0);
  d.num_blocks = nb, d.num_seqs = seqs, d.max_blocks = width, d.num_rows = rows;
  d.num_heads = static_cast<int32_t>(nh), d.head_dim = static_cast<int32_t>(hd), d.block_size = static_cast<int32_t>(bs);
  d.dtype = float_code(kind);
  return d;
}
// An expanded axis has several results at one place.
void separate(const char* name, const char* what, const at::Tensor& t) {
  for (int64_t i = 0; i < t.dim(); ++i)
    if (t.size(i) > 1 && t.stride(i) == 0) refuse(name, what, " must not be expanded");
}
at::Tensor paged_workspace(const at::Device& device, cudaStream_t stream) {
  static auto* spaces = new Workspaces();
  return workspace(*spaces, lib.paged_workspace_bytes(), device, stream);
}
int32_t count_of(const char* name, const char* what, PyObject* o) {
  const int64_t v = integer(name, what, o);
  if (v < 0) refuse(name, what, " must not be negative, got ", v);
  return static_cast<int32_t>(std::min<int64_t>(v, 0x7fffffff));
}
float scale_of(const char* name, PyObject* o, int64_t head_dim) {
  if (o == Py_None) return static_cast<float>(1.0 / std::sqrt(static_cast<double>(head_dim)));
  const double scale = PyFloat_AsDouble(o);
  if (scale == -1.0 && PyErr_Occurred()) throw python_error();
  if (!std::isfinite(static_cast<float>(scale) * 1.4426950408889634f)) refuse(name, "scale must be finite, in 32 bits and times log2 e");
  return static_cast<float>(scale);
}

// q, key_cache, value_cache, block_tables, context_lens, cu_seqlens, parents (None: a window), window, sinks, scale,
// return_lse, out
PyObject* py_paged(PyObject*, Args a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    const bool tree = n == 12 && a[6] != Py_None;
    const char* name = tree ? "paged_attention_tree" : "paged_attention_window";
    count(name, n, 12);
    const at::Tensor& q0 = tensor(name, "q", a[0]);
    Device dev{name};
    mak_paged_attn_desc d = {};
    d.window = count_of(name, "window", a[7]), d.sinks = count_of(name, "sinks", a[8]);
    if (d.sinks > 0 && d.window == 0) refuse(name, "sinks need a window");
    const bool want_lse = truth(a[10]), given = a[11] != Py_None;
    Used used;
    d.cache = paged_desc(name, a + 1, true, a[5], q0, used);
    const int64_t rows = q0.size(0), hq = q0.size(1), hd = q0.size(2);
    if (tree) {
      const at::Tensor& up = tensor(name, "parents", a[6]);
      if (up.dim() != 1 || up.size(0) != rows || up.scalar_type() != at::kInt) refuse(name, "parents must be int32 [rows]");
      if (!up.is_contiguous()) refuse(name, "parents must be contiguous");
      used.push_back(&up);
      d.parents = static_cast<const int32_t*>(up.data_ptr());
    }
    if (given) {
      const at::Tensor& o = tensor(name, "out", a[11]);
      if (o.sizes() != q0.sizes() || o.scalar_type() != q0.scalar_type() || (o.numel() && o.stride(2) != 1))
        refuse(name, "out must have q's shape and dtype and contiguous rows");
      separate(name, "out", o);
      used.push_back(&o);
    }
    d.scale = scale_of(name, a[9], hd);
    for (const at::Tensor* t : used) dev.add(*t);
    dev.need_library();
    const c10::cuda::CUDAGuard on(static_cast<c10::DeviceIndex>(dev.index));
    const at::Tensor q = aligned_rows(q0);
    const at::Tensor out = given ? THPVariable_Unpack(a[11]) : empty({rows, hq, hd}, q0.scalar_type(), q0.device());
    const at::Tensor lse = want_lse ? empty({rows, hq}, at::kFloat, q0.device()) : at::Tensor();
    const cudaStream_t stream = stream_of(dev);
    const at::Tensor ws = paged_workspace(q0.device(), stream);
    d.q = q.data_ptr(), d.out = out.data_ptr(), d.lse = want_lse ? static_cast<float*>(lse.data_ptr()) : nullptr;
    d.workspace = ws.data_ptr(), d.workspace_bytes = ws.numel();
    d.q_stride_row = q.stride(0), d.q_stride_head = q.stride(1), d.out_stride_row = out.stride(0), d.out_stride_head = out.stride(1);
    d.num_q_heads = static_cast<int32_t>(hq);
    check(lib.paged_attention(&d, stream), name);
    trace(name, a[0], "sm100a paged cache attention");
    return want_lse ? wrap(out, lse) : wrap(out);
  });
}

// q, key_cache, block_tables, context_lens, lse, sums, cu_seqlens, rows, window, sinks, scale, accumulate
PyObject* py_weights(PyObject*, Args a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    const char* name = "paged_attention_weights";
    count(name, n, 12);
    const at::Tensor &q0 = tensor(name, "q", a[0]), &lse = tensor(name, "lse", a[4]), &sums = tensor(name, "sums", a[5]);
    Device dev{name};
    mak_paged_weights_desc d = {};
    d.window = count_of(name, "window", a[8]), d.sinks = count_of(name, "sinks", a[9]);
    if (d.sinks > 0 && d.window == 0) refuse(name, "sinks need a window");
    d.accumulate = truth(a[11]);
    Used used;
    d.cache = paged_desc(name, a + 1, false, a[6], q0, used);
    const int64_t rows = q0.size(0), hq = q0.size(1), seqs = d.cache.num_seqs;
    if (lse.dim() != 2 || lse.size(0) != rows || lse.size(1) != hq || lse.scalar_type() != at::kFloat)
      refuse(name, "lse must be float32 [rows, num_q_heads]");
    if (hq > 1 && lse.stride(1) != 1) refuse(name, "a row of lse must be contiguous");
    if (sums.dim() != 3 || sums.size(1) != d.cache.num_heads || sums.scalar_type() != at::kFloat)
      refuse(name, "sums must be float32 [rows of sums, num_heads, max_tokens]");
    if (sums.size(2) > 1 && sums.stride(2) != 1) refuse(name, "the last axis of sums must be contiguous");
    separate(name, "sums", sums);
    if (a[7] == Py_None) {
      if (sums.size(0) != seqs) refuse(name, "without rows every sequence has its row of sums: ", sums.size(0), " rows for ", seqs, " sequences");
    } else {
      const at::Tensor& r = tensor(name, "rows", a[7]);
      if (r.dim() != 1 || r.size(0) != seqs || r.scalar_type() != at::kInt) refuse(name, "rows must be int32 [num_seqs]");
      if (!r.is_contiguous()) refuse(name, "rows must be contiguous");
      used.push_back(&r);
      d.rows = static_cast<const int32_t*>(r.data_ptr());
    }
    used.push_back(&lse);
    used.push_back(&sums);
    d.scale = scale_of(name, a[10], q0.size(2));
    for (const at::Tensor* t : used) dev.add(*t);
    dev.need_library();
    const c10::cuda::CUDAGuard on(static_cast<c10::DeviceIndex>(dev.index));
    // an expanded axis has no place in a tensor map
    const bool repeats = (rows > 1 && q0.stride(0) == 0) || (hq > 1 && q0.stride(1) == 0);
    const at::Tensor q = repeats ? q0.clone(at::MemoryFormat::Contiguous) : aligned_rows(q0);
    d.q = q.data_ptr(), d.lse = static_cast<const float*>(lse.data_ptr()), d.sums = static_cast<float*>(sums.data_ptr());
    d.q_stride_row = q.stride(0), d.q_stride_head = q.stride(1), d.lse_stride_row = lse.stride(0);
    d.sum_stride_row = sums.stride(0), d.sum_stride_head = sums.stride(1), d.sum_rows = sums.size(0), d.max_tokens = sums.size(2);
    d.num_q_heads = static_cast<int32_t>(hq);
    const cudaStream_t stream = stream_of(dev);
    const at::Tensor ws = paged_workspace(q0.device(), stream);
    d.workspace = ws.data_ptr(), d.workspace_bytes = ws.numel();
    check(lib.paged_weights(&d, stream), name);
    trace(name, a[0], "sm100a paged cache attention weights");
    Py_RETURN_NONE;
  });
}

// block_tables, context_lens, rows, ref_counts, key_caches, value_caches, sums, keep, sinks, recent
PyObject* py_evict(PyObject*, Args a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    const char* name = "kv_pages_evict";
    count(name, n, 10);
    const at::Tensor &table = tensor(name, "block_tables", a[0]), &lens = tensor(name, "context_lens", a[1]);
    const at::Tensor &rows = tensor(name, "rows", a[2]), &refs = tensor(name, "ref_counts", a[3]), &sums = tensor(name, "sums", a[6]);
    Device dev{name};
    mak_evict_desc e = {};
    e.keep = count_of(name, "keep", a[7]), e.sinks = count_of(name, "sinks", a[8]), e.recent = count_of(name, "recent", a[9]);
    if (e.keep < 1 || static_cast<int64_t>(e.sinks) + e.recent > e.keep) refuse(name, "keep must be at least 1 and sinks + recent");
    struct Held {
      std::vector<uint64_t> at;
      std::vector<const at::Tensor*> tensors;
      PyObject* list = nullptr;
      ~Held() { Py_XDECREF(list); }
    } held[2];
    const at::Tensor* first = nullptr;
    for (int which = 0; which < 2; ++which) {
      const char* what = which ? "value_caches" : "key_caches";
      Held& h = held[which];
      h.list = PySequence_Fast(a[4 + which], "key_caches and value_caches must be sequences of tensors");
      if (h.list == nullptr) throw python_error();
      for (Py_ssize_t i = 0; i < PySequence_Fast_GET_SIZE(h.list); ++i) {
        const at::Tensor& t = tensor(name, what, PySequence_Fast_GET_ITEM(h.list, i));
        if (t.dim() != 4) refuse(name, what, " must be [num_blocks, block_size, num_heads, head_dim]");
        if (first == nullptr) first = &t;
        if (t.sizes() != first->sizes() || t.scalar_type() != first->scalar_type()) refuse(name, "all caches must have one shape and type");
        if (!h.tensors.empty() && t.strides() != h.tensors[0]->strides()) refuse(name, what, " must have one layout");
        if (t.stride(3) != 1) refuse(name, "the head_dim axis of the caches must be contiguous");
        for (int x = 0; x < 3; ++x)
          if (t.size(x) > 1 && t.stride(x) % 8) refuse(name, "block, token and head strides of the caches must be multiples of 8 elements");
        if (reinterpret_cast<uintptr_t>(t.data_ptr()) % 16) refuse(name, "caches must begin on 16 bytes");
        h.at.push_back(reinterpret_cast<uintptr_t>(t.data_ptr()));
        h.tensors.push_back(&t);
      }
    }
    const int64_t layers = static_cast<int64_t>(held[0].at.size());
    if (layers != static_cast<int64_t>(held[1].at.size())) refuse(name, "key_caches and value_caches must have the same length");
    if (layers == 0) refuse(name, "key_caches must have a layer");
    if (first->scalar_type() != at::kHalf && first->scalar_type() != at::kBFloat16) refuse(name, "caches must be float16 or bfloat16");
    const int64_t nb = first->size(0), bs = first->size(1), nh = first->size(2), hd = first->size(3);
    if (hd != 64 && hd != 128 && hd != 256) refuse(name, "head_dim must be one of (64, 128, 256), got ", hd);
    if (nh < 1) refuse(name, "a cache needs heads");
    const mak_pages_desc d = pool(name, table, &lens, refs, bs, dev);
    if (refs.size(0) != nb) refuse(name, "ref_counts must have one entry per page of the caches");
    const int32_t* r = index_of(name, "rows", rows, 1, dev);
    if (sums.dim() != 4 || sums.size(0) != layers || sums.size(1) != table.size(0) || sums.size(2) != nh || sums.scalar_type() != at::kFloat)
      refuse(name, "sums must be float32 [layers, rows of block_tables, num_heads, max_tokens]");
    if (sums.size(3) > 1 && sums.stride(3) != 1) refuse(name, "the last axis of sums must be contiguous");
    separate(name, "sums", sums);
    for (int which = 0; which < 2; ++which) {
      const char* what = which ? "value_caches" : "key_caches";
      separate(name, what, *held[which].tensors[0]);  // one layout for all
      std::vector<uint64_t> sorted = held[which].at;
      std::sort(sorted.begin(), sorted.end());
      if (nb > 0 && std::adjacent_find(sorted.begin(), sorted.end()) != sorted.end()) refuse(name, what, " must not hold a layer twice");
    }
    for (const at::Tensor* t : {&table, &lens, &rows, &refs, &sums}) dev.add(*t);
    for (const Held& h : held)
      for (const at::Tensor* t : h.tensors) dev.add(*t);
    dev.need_library();
    const c10::cuda::CUDAGuard on(static_cast<c10::DeviceIndex>(dev.index));
    auto step = [&](const at::Tensor& c, int axis) { return c.size(axis) > 1 ? c.stride(axis) : nh * hd * bs; };
    const at::Tensor &kc = *held[0].tensors[0], &vc = *held[1].tensors[0];
    e.keys = held[0].at.data(), e.values = held[1].at.data(), e.sums = static_cast<float*>(sums.data_ptr());
    e.key_stride_block = step(kc, 0), e.key_stride_token = step(kc, 1), e.key_stride_head = step(kc, 2);
    e.value_stride_block = step(vc, 0), e.value_stride_token = step(vc, 1), e.value_stride_head = step(vc, 2);
    e.sum_stride_layer = sums.stride(0), e.sum_stride_row = sums.stride(1), e.sum_stride_head = sums.stride(2);
    e.num_layers = layers, e.max_tokens = sums.size(3), e.num_heads = static_cast<int32_t>(nh), e.head_dim = static_cast<int32_t>(hd);
    const int64_t want = rows.size(0);
    const at::Tensor room = empty({want + 1}, at::kInt, table.device());  // the answer and the scratch in one allocation
    int32_t* at = static_cast<int32_t*>(room.data_ptr());
    check(lib.evict(&d, &e, r, want, at, at + 1, stream_of(dev)), name);
    trace(name, a[0], "sm100a page eviction");
    return wrap(room.narrow(0, 0, 1));
  });
}

// ---- norms of q and k with the position rotation ----------------------------------------------------------

struct NormArgs {
  at::Tensor q, k, wq, wk, pos, cos, sin;
  double eps;
  bool interleaved;
};
// q, k, q_weight, k_weight, positions, cos, sin, eps, interleaved
NormArgs norm_args(const char* name, Args a) {
  NormArgs x{tensor(name, "q", a[0]), tensor(name, "k", a[1]), tensor(name, "q_weight", a[2]), tensor(name, "k_weight", a[3]),
             tensor(name, "positions", a[4]), tensor(name, "cos", a[5]), tensor(name, "sin", a[6]), 0.0, false};
  x.eps = PyFloat_AsDouble(a[7]);
  if (x.eps == -1.0 && PyErr_Occurred()) throw python_error();
  x.interleaved = truth(a[8]);
  return x;
}
mak_qk_norm_rope_desc norm_desc(const char* name, const NormArgs& x) {
  const at::Tensor &q = x.q, &k = x.k;
  if (q.dim() != 3 || k.dim() != 3 || q.size(0) != k.size(0) || q.size(2) != k.size(2))
    refuse(name, "q and k must be [tokens, heads, head_dim] with the same tokens and head_dim");
  const at::ScalarType kind = q.scalar_type();
  if ((kind != at::kHalf && kind != at::kBFloat16) || k.scalar_type() != kind) refuse(name, "q and k must both be float16 or both bfloat16");
  const int64_t tokens = q.size(0), hd = q.size(2);
  if (hd < 16 || hd > 256 || hd % 16) refuse(name, "head_dim must be a multiple of 16 up to 256, got ", hd);
  for (const at::Tensor* w : {&x.wq, &x.wk})
    if (w->dim() != 1 || w->size(0) != hd || (w->scalar_type() != at::kFloat && w->scalar_type() != kind) || w->scalar_type() != x.wq.scalar_type())
      refuse(name, "weights must both be [head_dim] in float32 or in q's type");
  if (x.pos.dim() != 1 || x.pos.size(0) != tokens || (x.pos.scalar_type() != at::kInt && x.pos.scalar_type() != at::kLong))
    refuse(name, "positions must be int32 or int64 [tokens]");
  if (x.cos.dim() != 2 || x.cos.sizes() != x.sin.sizes() || x.cos.scalar_type() != at::kFloat || x.sin.scalar_type() != at::kFloat)
    refuse(name, "cos and sin must both be float32 [max_positions, pairs]");
  const int64_t pairs = x.cos.size(1);
  if (pairs % 8 || 2 * pairs > hd) refuse(name, "the tables must have a multiple of 8 pairs, at most head_dim / 2, got ", pairs);
  if (!(x.eps >= 0.0)) refuse(name, "eps must not be negative");
  mak_qk_norm_rope_desc d = {};
  d.interleaved = x.interleaved, d.eps = static_cast<float>(x.eps);
  d.tokens = tokens, d.max_positions = x.cos.size(0);
  d.q_heads = static_cast<int32_t>(q.size(1)), d.k_heads = static_cast<int32_t>(k.size(1)), d.head_dim = static_cast<int32_t>(hd);
  d.rot_dim = static_cast<int32_t>(2 * pairs), d.dtype = float_code(kind), d.weight_dtype = float_code(x.wq.scalar_type());
  d.pos_dtype = x.pos.scalar_type() == at::kInt ? MAK_DT_I32 : MAK_DT_I64;
  return d;
}
void norm_on(Device& dev, const NormArgs& x) {
  for (const at::Tensor* t : {&x.q, &x.k, &x.wq, &x.wk, &x.pos, &x.cos, &x.sin}) dev.add(*t);
  dev.need_library();
}
// Copies where a layout needs one, on the device that is current by now.
void norm_inputs(mak_qk_norm_rope_desc& d, NormArgs& x) {
  x.q = aligned_rows(x.q), x.k = aligned_rows(x.k);
  x.wq = x.wq.contiguous(), x.wk = x.wk.contiguous(), x.pos = x.pos.contiguous();
  if (x.cos.stride(1) != 1) x.cos = x.cos.contiguous();
  if (x.sin.stride(1) != 1) x.sin = x.sin.contiguous();
  d.q = x.q.data_ptr(), d.k = x.k.data_ptr(), d.q_weight = x.wq.data_ptr(), d.k_weight = x.wk.data_ptr();
  d.positions = x.pos.data_ptr(), d.cos = static_cast<const float*>(x.cos.data_ptr()), d.sin = static_cast<const float*>(x.sin.data_ptr());
  d.q_stride_token = x.q.stride(0), d.q_stride_head = x.q.stride(1), d.k_stride_token = x.k.stride(0), d.k_stride_head = x.k.stride(1);
  d.cos_stride = x.cos.stride(0), d.sin_stride = x.sin.stride(0);
  d.qo_stride_token = static_cast<int64_t>(d.q_heads) * d.head_dim, d.ko_stride_token = static_cast<int64_t>(d.k_heads) * d.head_dim;
  d.qo_stride_head = d.ko_stride_head = d.head_dim;
}

std::array<at::Tensor, 2> norm_forward(NormArgs x) {
  const char* name = "apply_qk_norm_rope";
  Device dev{name};
  mak_qk_norm_rope_desc d = norm_desc(name, x);
  norm_on(dev, x);
  const c10::cuda::CUDAGuard on(static_cast<c10::DeviceIndex>(dev.index));
  norm_inputs(d, x);
  const at::ScalarType kind = x.q.scalar_type();
  std::array<at::Tensor, 2> y = {empty(x.q.sizes(), kind, x.q.device()), empty(x.k.sizes(), kind, x.q.device())};
  d.q_out = y[0].data_ptr(), d.k_out = y[1].data_ptr();
  check(lib.norm_rope(&d, stream_of(dev)), name);
  return y;
}

std::array<at::Tensor, 4> norm_backward(const at::Tensor& gq0, const at::Tensor& gk0, NormArgs x) {
  const char* name = "apply_qk_norm_rope_backward";
  Device dev{name};
  mak_qk_norm_rope_desc d = norm_desc(name, x);
  if (gq0.sizes() != x.q.sizes() || gk0.sizes() != x.k.sizes() || gq0.scalar_type() != x.q.scalar_type() || gk0.scalar_type() != x.q.scalar_type())
    refuse(name, "grad_q and grad_k must have the shapes and type of q and k");
  dev.add(gq0);
  dev.add(gk0);
  norm_on(dev, x);
  const c10::cuda::CUDAGuard on(static_cast<c10::DeviceIndex>(dev.index));
  norm_inputs(d, x);
  const at::Tensor gq = aligned_rows(gq0), gk = aligned_rows(gk0);
  const at::ScalarType kind = x.q.scalar_type(), weight = x.wq.scalar_type();
  std::array<at::Tensor, 4> got = {empty(x.q.sizes(), kind, x.q.device()), empty(x.k.sizes(), kind, x.q.device()),
                                   empty(x.wq.sizes(), weight, x.q.device()), empty(x.wk.sizes(), weight, x.q.device())};
  const at::Tensor partial = empty({lib.norm_partial(d.head_dim)}, at::kFloat, x.q.device());
  // a tensor without elements has no address, but the call is still a backward one
  static float none[4];
  auto address = [](const at::Tensor& t) { return t.numel() ? t.data_ptr() : static_cast<void*>(none); };
  d.grad_q = address(gq), d.grad_k = address(gk);
  d.gq_stride_token = gq.stride(0), d.gq_stride_head = gq.stride(1), d.gk_stride_token = gk.stride(0), d.gk_stride_head = gk.stride(1);
  d.q_out = got[0].data_ptr(), d.k_out = got[1].data_ptr(), d.grad_q_weight = got[2].data_ptr(), d.grad_k_weight = got[3].data_ptr();
  d.partial = static_cast<float*>(partial.data_ptr());
  check(lib.norm_rope(&d, stream_of(dev)), name);
  return got;
}

// The node of a call whose q, k or weights want a gradient.
struct NormNode : torch::autograd::Function<NormNode> {
  using Context = torch::autograd::AutogradContext;
  using List = torch::autograd::variable_list;
  static List forward(Context* ctx, const at::Tensor& q, const at::Tensor& k, const at::Tensor& wq, const at::Tensor& wk, const at::Tensor& pos,
                      const at::Tensor& cos, const at::Tensor& sin, double eps, bool interleaved) {
    ctx->save_for_backward({q, k, wq, wk, pos, cos, sin});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["interleaved"] = interleaved;
    const auto y = norm_forward({q, k, wq, wk, pos, cos, sin, eps, interleaved});
    return {y[0], y[1]};
  }
  // Runs on a thread of autograd's: only exceptions of the standard library may leave it.
  static List backward(Context* ctx, List grads) {
    const List s = ctx->get_saved_variables();
    List got;
    try {
      no_tangent("apply_qk_norm_rope", {&grads[0], &grads[1]});
      const auto g = norm_backward(grads[0], grads[1], {s[0], s[1], s[2], s[3], s[4], s[5], s[6], ctx->saved_data["eps"].toDouble(),
                                                        ctx->saved_data["interleaved"].toBool()});
      got.assign(g.begin(), g.end());
    } catch (const Refused& r) {
      TORCH_CHECK(false, r.text);
    }
    if (c10::GradMode::is_enabled()) {  // a graph of the gradient is wanted: it ends here, in an error when it is walked
      for (at::Tensor& t : got) t.set_requires_grad(true);
      got = std::make_shared<torch::autograd::DelayedError>("apply_qk_norm_rope: the gradient has no gradient of its own", 4)->apply(std::move(got));
    }
    got.resize(9);
    return got;
  }
};

// the nine of norm_args
PyObject* py_norm(PyObject*, Args a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    const char* name = "apply_qk_norm_rope";
    count(name, n, 9);
    const NormArgs x = norm_args(name, a);
    no_tangent(name, {&x.q, &x.k, &x.wq, &x.wk, &x.cos, &x.sin});
    bool wants = false;
    if (c10::GradMode::is_enabled()) {
      if (x.cos.requires_grad() || x.sin.requires_grad()) refuse(name, "cos and sin are tables without a gradient, detach them");
      for (const at::Tensor* t : {&x.q, &x.k, &x.wq, &x.wk}) wants = wants || t->requires_grad();
    }
    PyObject* got;
    if (wants) {
      const auto y = NormNode::apply(x.q, x.k, x.wq, x.wk, x.pos, x.cos, x.sin, x.eps, x.interleaved);
      got = wrap(y[0], y[1]);
    } else {
      const auto y = norm_forward(x);
      got = wrap(y[0], y[1]);
    }
    trace(name, a[0], "sm100a norms and rotary positions");
    return got;
  });
}

// grad_q, grad_k, the nine of norm_args
PyObject* py_norm_back(PyObject*, Args a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    const char* name = "apply_qk_norm_rope_backward";
    count(name, n, 11);
    const auto got = norm_backward(tensor(name, "grad_q", a[0]), tensor(name, "grad_k", a[1]), norm_args(name, a + 2));
    trace(name, a[0], "sm100a gradient of norms and rotary positions");
    PyObject* all = PyTuple_New(4);
    if (all == nullptr) throw python_error();
    for (int i = 0; i < 4; ++i) PyTuple_SET_ITEM(all, i, THPVariable_Wrap(got[i]));
    return all;
  });
}

// ---- the module -----------------------------------------------------------------------------------------------

// bind(addresses: dict of name -> int, emit): the library's entry points and the trace function
PyObject* py_bind(PyObject*, Args a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    count("bind", n, 2);
    auto at = [&](const char* name) {
      PyObject* v = PyDict_GetItemString(a[0], name);
      if (v == nullptr) throw Refused{cat("bind: no address of ", name), true};
      void* p = PyLong_AsVoidPtr(v);
      if (p == nullptr) throw Refused{cat("bind: no address of ", name), true};
      return p;
    };
#define MAK_BIND(FIELD, NAME) lib.FIELD = reinterpret_cast<decltype(lib.FIELD)>(at(#NAME))
    MAK_BIND(last_error, mak_last_error);
    MAK_BIND(workspace_bytes, mak_block_attention_workspace_bytes);
    MAK_BIND(append, mak_block_append);
    MAK_BIND(fork, mak_pages_fork);
    MAK_BIND(grow, mak_pages_grow);
    MAK_BIND(free, mak_pages_free);
    MAK_BIND(compact, mak_pages_compact);
    MAK_BIND(copy, mak_pages_copy);
    MAK_BIND(rope, mak_rope_axes);
    MAK_BIND(paged_workspace_bytes, mak_paged_attention_workspace_bytes);
    MAK_BIND(paged_attention, mak_paged_attention);
    MAK_BIND(paged_weights, mak_paged_weights);
    MAK_BIND(evict, mak_pages_evict);
    MAK_BIND(norm_partial, mak_qk_norm_rope_partial_floats);
    MAK_BIND(norm_rope, mak_qk_norm_rope);
    MAK_BIND(attention, mak_block_attention);
#undef MAK_BIND
    Py_INCREF(a[1]);
    Py_XDECREF(emit);
    emit = a[1];
    Py_RETURN_NONE;
  });
}

#define MAK_FAST(F) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(F)), METH_FASTCALL, nullptr
PyMethodDef methods[] = {{"bind", MAK_FAST(py_bind)},       {"attend", MAK_FAST(py_attend)}, {"append", MAK_FAST(py_append)},
                         {"fork", MAK_FAST(py_fork)},       {"grow", MAK_FAST(py_grow)},     {"free", MAK_FAST(py_free)},
                         {"compact", MAK_FAST(py_compact)}, {"copy", MAK_FAST(py_copy)},     {"rope", MAK_FAST(py_rope)},
                         {"paged", MAK_FAST(py_paged)},     {"weights", MAK_FAST(py_weights)}, {"evict", MAK_FAST(py_evict)},
                         {"norm", MAK_FAST(py_norm)},       {"norm_back", MAK_FAST(py_norm_back)},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_mak_front", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject* PyInit__mak_front() { return PyModule_Create(&module); }
