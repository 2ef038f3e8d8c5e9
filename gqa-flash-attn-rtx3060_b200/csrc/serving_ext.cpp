// Python binding of the ragged serving step (module gqa_kernels._serving_ext).
//
// A step makes these calls for every layer, so what a call costs on the host matters as
// much as the kernel for small batches: argument checks, output allocation, the
// workspace and the call of the C ABI (include/gqa_sm100.h) are done here in one go, a
// few microseconds instead of the ten that the same checks take in Python. The library
// itself stays behind its C ABI: its entry points are bound by address (bind()), so that
// the release and the checked library both work.
//
// Checks come in the order shapes, types, values, device, so that all but the last can be
// tested on a machine without a GPU. C++ exceptions do not leave an entry point.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <cuda_runtime_api.h>
#include <torch/csrc/autograd/python_variable.h>

#include <atomic>
#include <cmath>
#include <climits>
#include <map>
#include <mutex>
#include <stdexcept>
#include <string>
#include <utility>
#include <vector>

#include "gqa_sm100.h"

namespace {

struct PyError {};  // a Python exception is set

[[noreturn]] void fail(PyObject* type, const char* text) {
  PyErr_SetString(type, text);
  throw PyError{};
}
#define CHECK_VALUE(cond, text) \
  do {                          \
    if (!(cond)) fail(PyExc_ValueError, text); \
  } while (0)
#define CHECK_TYPE(cond, text) \
  do {                         \
    if (!(cond)) fail(PyExc_TypeError, text); \
  } while (0)

// ----------------------------------------------------------------------------- the library
struct Library {
  int (*step_plan)(const gqa_step_plan_args*, void*) = nullptr;
  int (*rope)(const gqa_qk_norm_rope_args*, void*) = nullptr;
  int (*ragged)(const gqa_ragged_args*, void*) = nullptr;
  size_t (*ragged_bytes)(const gqa_ragged_args*) = nullptr;
  int (*verify)(const gqa_verify_args*, void*) = nullptr;
  int (*greedy)(const gqa_verify_args*, void*) = nullptr;
  size_t (*verify_bytes)(const gqa_verify_args*, int) = nullptr;
  const char* (*strerror)(int) = nullptr;
} g_lib;

void check_status(int rc, const char* what) {
  if (rc == GQA_OK) return;
  PyErr_Format(PyExc_RuntimeError, "%s failed: %s (status %d)", what, g_lib.strerror(rc), rc);
  throw PyError{};
}

// ----------------------------------------------------------------------------- arguments
const at::Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) {
    PyErr_Format(PyExc_TypeError, "%s must be a tensor", name);
    throw PyError{};
  }
  return THPVariable_Unpack(o);
}
// A tensor, or an undefined one for None.
at::Tensor optional(PyObject* o, const char* name) { return o == Py_None ? at::Tensor() : tensor(o, name); }

long long integer(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw PyError{};
  return v;
}
int integer32(PyObject* o, const char* text) {
  const long long v = integer(o);
  CHECK_VALUE(v >= INT_MIN && v <= INT_MAX, text);
  return (int)v;
}
double number(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw PyError{};
  return v;
}
bool truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw PyError{};
  return v != 0;
}

int dtype16(const at::Tensor& t) {
  if (t.scalar_type() == at::kBFloat16) return GQA_DTYPE_BF16;
  if (t.scalar_type() == at::kHalf) return GQA_DTYPE_F16;
  PyErr_Format(PyExc_RuntimeError, "gqa_kernels supports float16 and bfloat16 tensors, got %s", c10::toString(t.scalar_type()));
  throw PyError{};
}
bool is(const at::Tensor& t, at::ScalarType s) { return t.scalar_type() == s; }
bool shaped(const at::Tensor& t, std::initializer_list<int64_t> s) { return t.sizes() == at::IntArrayRef(s); }
int dim32(const at::Tensor& t, int i) {
  CHECK_VALUE(t.size(i) <= INT_MAX, "a dimension is too large");
  return (int)t.size(i);
}

// All defined tensors on one CUDA device, whose index is returned.
int device_of(std::initializer_list<const at::Tensor*> ts) {
  int index = -1;
  for (const at::Tensor* t : ts) {
    if (!t->defined()) continue;
    CHECK_VALUE(t->is_cuda(), "tensors must be on a CUDA device");
    if (index < 0) index = t->get_device();
    CHECK_VALUE(t->get_device() == index, "tensors must be on one device");
  }
  return index;
}

// Rows that the kernels read in 16-byte pieces: d stride 1, the others multiples of
// `multiple`, base 16-byte aligned; other layouts are copied once. (contiguous() would not
// copy a tensor that is contiguous on another base.) A dimension of size 1 may have any
// stride, since no element lies a stride away.
bool rows_ok(const at::Tensor& t, int64_t multiple) {
  const int64_t n = t.dim();
  if (t.stride(n - 1) != 1 && t.size(n - 1) != 1) return false;
  if (reinterpret_cast<uintptr_t>(t.const_data_ptr()) & 15) return false;
  for (int64_t i = 0; i + 1 < n; ++i)
    if (t.size(i) != 1 && (t.stride(i) % multiple != 0 || t.stride(i) < 0)) return false;
  return true;
}
at::Tensor rows(const at::Tensor& t) { return rows_ok(t, 8) ? t : t.clone(at::MemoryFormat::Contiguous); }
at::Tensor flat(const at::Tensor& t) { return !t.defined() || t.is_contiguous() ? t : t.contiguous(); }
bool last_dim_ok(const at::Tensor& t) { return t.stride(-1) == 1 || t.size(-1) <= 1; }
// The strides that the library gets, a dimension of size 1 as if it were contiguous.
void strides_of(const at::Tensor& t, int64_t* out) {
  int64_t next = 1;
  for (int64_t i = t.dim() - 1; i >= 0; --i) {
    out[i] = t.size(i) == 1 ? next : t.stride(i);
    next = out[i] * t.size(i);
  }
}
template <typename T>
T* data(const at::Tensor& t) {
  return t.defined() ? reinterpret_cast<T*>(t.data_ptr()) : nullptr;
}
at::Tensor empty(at::IntArrayRef sizes, at::ScalarType dtype, int device) {
  return at::detail::empty_cuda(sizes, dtype, c10::Device(c10::kCUDA, (c10::DeviceIndex)device), std::nullopt);
}

// ----------------------------------------------------------------------------- workspaces
// One per (device, stream); its counters have the same place for every call, so nothing is
// zeroed after its allocation, and it only grows. Every one ever handed out is kept: a call
// that took it may still be queued.
//
// A stream that is being captured has another one for as long as that capture lasts: its
// counters are zeroed by the graph, before its first call, so that every replay starts from
// zero whatever ran before it (other graphs of the same stream, or a replay that an expired
// wait ended). It lives as long as the graph, and replays of different graphs may overlap.
struct Workspace {
  void* ptr = nullptr;
  size_t bytes = 0;
};
struct CapturedWorkspace {
  unsigned long long capture = 0;  // ids are not reused
  Workspace ws;
};
std::map<std::pair<int, void*>, Workspace> g_workspaces;
std::map<std::pair<int, void*>, CapturedWorkspace> g_captured;
std::vector<at::Tensor>* g_buffers = nullptr;  // never freed: the interpreter may be gone before it
std::mutex g_mutex;

// Buffers whose graphs are gone. The runtime says so on a thread of its own, from which
// no CUDA call may be made: a later call frees them.
std::vector<at::Tensor*>* g_gone = nullptr;
std::atomic<bool> g_any_gone{false};
std::mutex g_gone_mutex;

void CUDART_CB graph_gone(void* buffer) {
  std::lock_guard<std::mutex> lock(g_gone_mutex);
  if (!g_gone) g_gone = new std::vector<at::Tensor*>();
  g_gone->push_back(static_cast<at::Tensor*>(buffer));
  g_any_gone.store(true);
}
void free_gone() {
  std::vector<at::Tensor*> gone;
  {
    std::lock_guard<std::mutex> lock(g_gone_mutex);
    if (g_gone) gone.swap(*g_gone);
    g_any_gone.store(false);
  }
  for (at::Tensor* t : gone) delete t;
}

Workspace grow_workspace(int device, void* stream, size_t need) {
  std::lock_guard<std::mutex> lock(g_mutex);
  Workspace& ws = g_workspaces[{device, stream}];
  if (ws.bytes < need) {
    const size_t n = std::max<size_t>(std::max<size_t>(need, size_t(4) << 20), 2 * ws.bytes);
    at::Tensor buf = empty({(int64_t)n}, at::kByte, device);
    buf.zero_();
    if (!g_buffers) g_buffers = new std::vector<at::Tensor>();
    g_buffers->push_back(buf);
    ws = Workspace{buf.data_ptr(), n};
  }
  return ws;
}

void check_cuda(cudaError_t e, const char* what) {
  if (e == cudaSuccess) return;
  PyErr_Format(PyExc_RuntimeError, "%s failed: %s", what, cudaGetErrorString(e));
  throw PyError{};
}

// A workspace of at least `need` bytes for calls that are captured on `stream` into `graph`.
Workspace captured_workspace(int device, void* stream, unsigned long long capture, cudaGraph_t graph, size_t need) {
  std::lock_guard<std::mutex> lock(g_mutex);
  CapturedWorkspace& c = g_captured[{device, stream}];
  if (c.capture == capture && c.ws.bytes >= need) return c.ws;
  need = std::max<size_t>(need, GQA_SERVING_COUNTER_BYTES);
  auto* buf = new at::Tensor(empty({(int64_t)need}, at::kByte, device));
  cudaUserObject_t owner = nullptr;
  const cudaError_t e = cudaUserObjectCreate(&owner, buf, graph_gone, 1, cudaUserObjectNoDestructorSync);
  if (e != cudaSuccess) delete buf;
  check_cuda(e, "cudaUserObjectCreate");
  check_cuda(cudaGraphRetainUserObject(graph, owner, 1, cudaGraphUserObjectMove), "cudaGraphRetainUserObject");
  check_cuda(cudaMemsetAsync(buf->data_ptr(), 0, GQA_SERVING_COUNTER_BYTES, static_cast<cudaStream_t>(stream)), "cudaMemsetAsync");
  c = CapturedWorkspace{capture, Workspace{buf->data_ptr(), need}};
  return c.ws;
}

void drop_workspaces(int device) {
  std::lock_guard<std::mutex> lock(g_mutex);
  for (auto it = g_workspaces.begin(); it != g_workspaces.end();)
    it = it->first.first == device ? g_workspaces.erase(it) : std::next(it);
}

// Calls f(stream) on `device`, with that device current.
template <typename F>
void on_device(int device, const char* what, F f) {
  c10::cuda::OptionalCUDAGuard guard;
  if (c10::cuda::current_device() != device) guard.set_index((c10::DeviceIndex)device);
  check_status(f(c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream()), what);
}
template <typename A, typename F, typename N>
void with_workspace(int device, const char* what, A& args, F f, N need) {
  on_device(device, what, [&](cudaStream_t st) {
    cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
    unsigned long long capture = 0;
    cudaGraph_t graph = nullptr;
    check_cuda(cudaStreamGetCaptureInfo(st, &status, &capture, &graph), "cudaStreamGetCaptureInfo");
    if (status == cudaStreamCaptureStatusActive) {
      const Workspace ws = captured_workspace(device, st, capture, graph, need(&args));
      args.workspace = ws.ptr;
      args.workspace_bytes = ws.bytes;
      return f(&args, st);
    }
    if (g_any_gone.load(std::memory_order_relaxed)) free_gone();
    Workspace ws;
    {
      std::lock_guard<std::mutex> lock(g_mutex);
      auto it = g_workspaces.find({device, (void*)st});
      if (it != g_workspaces.end()) ws = it->second;
    }
    int rc = GQA_ERR_WORKSPACE;
    if (ws.ptr) {
      args.workspace = ws.ptr;
      args.workspace_bytes = ws.bytes;
      rc = f(&args, st);
    }
    if (rc == GQA_ERR_WORKSPACE) {
      ws = grow_workspace(device, st, need(&args));
      args.workspace = ws.ptr;
      args.workspace_bytes = ws.bytes;
      rc = f(&args, st);
    }
    // Anything but a refusal: the counters are not trusted any more.
    if (rc != GQA_OK && rc != GQA_ERR_INVALID_ARG && rc != GQA_ERR_UNSUPPORTED && rc != GQA_ERR_ALIGNMENT) drop_workspaces(device);
    return rc;
  });
}

// ----------------------------------------------------------------------------- step plan
// (query_lens, context_lens, block_tables, blocks_held, free_blocks, free_count, block_size,
//  max_tokens, cu, seq_lens, positions, slots, token_seqs, granted, held_out, free_out)
void step_plan(PyObject* const* a) {
  const at::Tensor &q = tensor(a[0], "query_lens"), &ctx = tensor(a[1], "context_lens"), &bt = tensor(a[2], "block_tables"),
                   &held = tensor(a[3], "blocks_held"), &fr = tensor(a[4], "free_blocks"), &fc = tensor(a[5], "free_count");
  const at::Tensor &cu = tensor(a[8], "cu_query_lens"), &sl = tensor(a[9], "seq_lens"), &pos = tensor(a[10], "positions"),
                   &slots = tensor(a[11], "slot_mapping"), &ts = tensor(a[12], "token_seqs"), &gr = tensor(a[13], "granted"),
                   &ho = tensor(a[14], "blocks_held"), &fo = tensor(a[15], "free_count");
  CHECK_VALUE(q.dim() == 1, "query_lens must be (n,)");
  const int64_t n = q.size(0);
  CHECK_VALUE(shaped(ctx, {n}) && shaped(held, {n}) && bt.dim() == 2 && bt.size(0) == n,
              "query_lens, context_lens and blocks_held must be (n,) and block_tables (n, max_blocks)");
  CHECK_VALUE(fr.dim() == 1 && shaped(fc, {1}), "free_blocks must be (num_free,) and free_count (1,)");
  for (const at::Tensor* t : {&q, &ctx, &bt, &held, &fr, &fc})
    CHECK_TYPE(is(*t, at::kInt), "lengths, tables and the free list must be int32");
  const long long block = integer(a[6]), max_tokens = integer(a[7]);
  CHECK_VALUE(block >= 1 && block <= (1 << 30) && (block & (block - 1)) == 0, "block_size must be a power of two");
  CHECK_VALUE(max_tokens >= 0 && max_tokens <= INT_MAX, "max_tokens must not be negative");
  const int64_t width = bt.size(1);
  CHECK_VALUE(bt.stride(1) == 1 || width <= 1, "the rows of block_tables must be contiguous");
  CHECK_VALUE(n <= 1 || bt.stride(0) >= width, "the rows of block_tables must not overlap");
  for (const at::Tensor* t : {&q, &ctx, &held, &fr})
    CHECK_VALUE(t->size(0) <= 1 || t->stride(0) == 1, "lengths and the free list must be contiguous");
  CHECK_VALUE(shaped(cu, {n + 1}) && shaped(sl, {n}) && shaped(pos, {max_tokens}) && shaped(slots, {max_tokens}) &&
                  shaped(ts, {max_tokens}) && shaped(gr, {n}) && shaped(ho, {n}) && shaped(fo, {1}) && is(cu, at::kInt) &&
                  is(sl, at::kInt) && is(pos, at::kInt) && is(slots, at::kLong) && is(ts, at::kInt) && is(gr, at::kBool) &&
                  is(ho, at::kInt) && is(fo, at::kInt),
              "out must be a StepPlan of this n and max_tokens");
  for (const at::Tensor* t : {&cu, &sl, &pos, &slots, &ts, &gr, &ho})
    CHECK_VALUE(t->size(0) <= 1 || t->stride(0) == 1, "out must be a StepPlan of contiguous tensors");
  const int device = device_of({&q, &ctx, &bt, &held, &fr, &fc, &cu, &sl, &pos, &slots, &ts, &gr, &ho, &fo});
  CHECK_VALUE(ho.data_ptr() != held.data_ptr() || n == 0, "out must not hold the tensors that the plan is made from");
  CHECK_VALUE(fo.data_ptr() != fc.data_ptr(), "out must not hold the tensors that the plan is made from");
  CHECK_VALUE(sl.data_ptr() != ctx.data_ptr() || n == 0, "out must not hold the tensors that the plan is made from");
  gqa_step_plan_args g{};
  g.query_lens = data<int>(q);
  g.context_lens = data<int>(ctx);
  g.block_tables = data<int>(bt);
  g.blocks_held = data<int>(held);
  g.free_blocks = data<int>(fr);
  g.free_count = data<int>(fc);
  g.cu_query_lens = data<int>(cu);
  g.seq_lens = data<int>(sl);
  g.positions = data<int>(pos);
  g.slot_mapping = data<int64_t>(slots);
  g.token_seqs = data<int>(ts);
  g.granted = data<unsigned char>(gr);
  g.blocks_held_out = data<int>(ho);
  g.free_count_out = data<int>(fo);
  g.bt_stride = std::max<int64_t>(n > 1 ? bt.stride(0) : 0, width);
  g.num_seqs = dim32(q, 0);
  g.max_blocks = dim32(bt, 1);
  g.num_free = dim32(fr, 0);
  g.block_size = (int)block;
  g.max_tokens = (int)max_tokens;
  on_device(device, "gqa_step_plan", [&](cudaStream_t st) { return g_lib.step_plan(&g, st); });
}

// ----------------------------------------------------------------------------- norm, rotation, cache write
// (q, k, v | None, positions, cos_sin, key_cache | None, value_cache | None, slots | None, q_weight |
//  None, k_weight | None, eps, sections | None, interleaved, out | None, k_scale, v_scale)
// Returns q, or without a cache (q, k).
PyObject* norm_rope(PyObject* const* a) {
  at::Tensor q = tensor(a[0], "q"), k = tensor(a[1], "k"), v = optional(a[2], "v");
  at::Tensor pos = tensor(a[3], "positions");
  const at::Tensor& table = tensor(a[4], "cos_sin");
  const at::Tensor kc = optional(a[5], "key_cache"), vc = optional(a[6], "value_cache");
  at::Tensor slots = optional(a[7], "slot_mapping");
  const at::Tensor qw = optional(a[8], "q_weight"), kw = optional(a[9], "k_weight");
  CHECK_VALUE(q.dim() == 3 && k.dim() == 3, "q and k must be (num_tokens, heads, head_dim)");
  const int64_t tokens = q.size(0), d = q.size(2), hkv = k.size(1);
  CHECK_VALUE(k.size(0) == tokens && k.size(2) == d, "q and k must have the same tokens and head_dim");
  CHECK_VALUE(d == 64 || d == 128, "unsupported head_dim: 64 or 128");
  gqa_qk_norm_rope_args g{};
  g.dtype = dtype16(q);
  CHECK_TYPE(k.scalar_type() == q.scalar_type(), "q and k must share one dtype");
  g.eps = (float)number(a[10]);
  g.k_scale = (float)number(a[14]);
  g.v_scale = (float)number(a[15]);
  const bool cached = kc.defined();
  CHECK_VALUE(cached || (!v.defined() && !vc.defined() && !slots.defined()),
              "the cache write needs key_cache, value_cache and slot_mapping");
  if (cached) {
    CHECK_VALUE(v.defined() && vc.defined() && slots.defined() && v.sizes() == k.sizes() && kc.dim() == 4 && vc.sizes() == kc.sizes() &&
                    kc.size(2) == hkv && kc.size(3) == d,
                "k/v must be (num_tokens, num_kv_heads, head_dim) and the caches (num_blocks, block_size, num_kv_heads, head_dim)");
    g.cache_fp8 = is(kc, at::kFloat8_e4m3fn);
    CHECK_TYPE(v.scalar_type() == k.scalar_type() && vc.scalar_type() == kc.scalar_type() &&
                   (g.cache_fp8 || kc.scalar_type() == k.scalar_type()),
               "k and v share q's dtype; the caches share it too, or are both float8_e4m3fn");
    CHECK_VALUE(kc.is_contiguous() && vc.is_contiguous(), "the caches must be contiguous");
    CHECK_TYPE(is(slots, at::kLong) && shaped(slots, {tokens}), "slot_mapping must be int64 (num_tokens,)");
    CHECK_VALUE(!g.cache_fp8 || (g.k_scale > 0 && g.v_scale > 0), "fp8 caches need positive k_scale and v_scale");
  }
  CHECK_VALUE(is(pos, at::kInt) && (pos.dim() == 1 || pos.dim() == 2) && pos.size(-1) == tokens,
              "positions must be int32 (num_tokens,) or (axes, num_tokens)");
  const int64_t axes = pos.dim() == 1 ? 1 : pos.size(0);
  CHECK_VALUE(axes >= 1 && axes <= 4, "1 to 4 position axes are supported");
  CHECK_VALUE(is(table, at::kFloat) && table.dim() == 2 && table.is_contiguous() &&
                  (reinterpret_cast<uintptr_t>(table.const_data_ptr()) & 15) == 0,
              "cos_sin must be a contiguous, 16-byte aligned float32 (max_positions, rotary_dim)");
  const int64_t rot = table.size(1);
  CHECK_VALUE(rot <= d && rot % 16 == 0, "rotary_dim must be a multiple of 16, at most head_dim");
  if (a[11] == Py_None) {
    CHECK_VALUE(axes == 1, "several position axes need sections");
    g.sections[0] = (int)(rot / 2);
  } else {
    PyObject* seq = PySequence_Fast(a[11], "sections must be a sequence of integers");
    if (!seq) throw PyError{};
    const bool count = PySequence_Fast_GET_SIZE(seq) == axes;
    long long sum = 0;
    bool fine = count;
    for (int64_t i = 0; count && i < axes; ++i) {
      const long long x = PyLong_AsLongLong(PySequence_Fast_GET_ITEM(seq, i));
      if (x == -1 && PyErr_Occurred()) {
        Py_DECREF(seq);
        throw PyError{};
      }
      fine = fine && x >= 0 && x <= rot;
      g.sections[i] = (int)x;
      sum += x;
    }
    Py_DECREF(seq);
    CHECK_VALUE(fine && sum * 2 == rot, "sections must give each position axis its share of the rotary_dim / 2 frequencies");
  }
  for (const at::Tensor* w : {&qw, &kw})
    CHECK_VALUE(!w->defined() || (shaped(*w, {d}) && w->scalar_type() == q.scalar_type() && w->stride(0) == 1 &&
                                  (reinterpret_cast<uintptr_t>(w->const_data_ptr()) & 15) == 0),
                "norm weights must be contiguous (head_dim,) tensors of q's dtype, 16-byte aligned");
  at::Tensor out = optional(a[13], "out");
  CHECK_VALUE(!out.defined() || (out.sizes() == q.sizes() && out.scalar_type() == q.scalar_type() && out.is_contiguous()),
              "out must be a contiguous tensor of q's shape and dtype");
  const int device = device_of({&q, &k, &v, &pos, &table, &kc, &vc, &slots, &qw, &kw, &out});
  if (!out.defined()) out = empty(q.sizes(), q.scalar_type(), device);
  at::Tensor k_out = cached ? kc : empty(k.sizes(), k.scalar_type(), device);
  q = rows(q);
  k = rows(k);
  if (cached) v = rows(v);
  if (pos.size(-1) > 1 && pos.stride(-1) != 1) pos = pos.contiguous();
  slots = flat(slots);
  g.q = q.data_ptr();
  g.k = k.data_ptr();
  g.v = cached ? v.data_ptr() : nullptr;
  g.q_weight = data<void>(qw);
  g.k_weight = data<void>(kw);
  g.positions = data<int>(pos);
  g.cos_sin = data<float>(table);
  g.q_out = out.data_ptr();
  g.k_dst = k_out.data_ptr();
  g.v_dst = data<void>(vc);
  g.slot_mapping = data<int64_t>(slots);
  strides_of(q, g.q_strides);
  strides_of(k, g.k_strides);
  if (cached) strides_of(v, g.v_strides);
  g.pos_stride = axes > 1 ? pos.stride(0) : 0;
  g.axes = (int)axes;
  g.max_positions = dim32(table, 0);
  g.rotary_dim = (int)rot;
  g.interleaved = truth(a[12]);
  g.num_tokens = dim32(q, 0);
  g.num_heads = dim32(q, 1);
  g.num_kv_heads = dim32(k, 1);
  g.head_dim = (int)d;
  g.block_size = cached ? dim32(kc, 1) : 0;
  g.num_blocks = cached ? dim32(kc, 0) : 0;
  on_device(device, "gqa_qk_norm_rope", [&](cudaStream_t st) { return g_lib.rope(&g, st); });
  PyObject* r = THPVariable_Wrap(out);
  if (cached) return r;
  PyObject* rk = THPVariable_Wrap(k_out);
  PyObject* both = PyTuple_Pack(2, r, rk);
  Py_XDECREF(r);
  Py_XDECREF(rk);
  return both;
}

// ----------------------------------------------------------------------------- ragged attention
// (query, key_cache, value_cache, block_tables, cu, seq_lens, max_query_len | None, max_seq_len | None,
//  scale | None, causal, softcap, alibi | None, window | None, prefix | None, key_starts | None,
//  k_scale, v_scale, return_lse, out | None)
PyObject* ragged(PyObject* const* a) {
  at::Tensor q = tensor(a[0], "query");
  const at::Tensor &kc = tensor(a[1], "key_cache"), &vc = tensor(a[2], "value_cache");
  at::Tensor bt = tensor(a[3], "block_tables"), cu = tensor(a[4], "cu_query_lens"), lens = tensor(a[5], "seq_lens");
  at::Tensor alibi = optional(a[11], "alibi_slopes"), prefix = optional(a[13], "prefix_lens"), starts = optional(a[14], "key_starts");
  CHECK_VALUE(q.dim() == 3 && kc.dim() == 4,
              "query must be (num_tokens, num_heads, head_dim) and the caches (num_blocks, block_size, num_kv_heads, head_dim)");
  const int64_t tokens = q.size(0), hq = q.size(1), d = q.size(2), hkv = kc.size(2);
  CHECK_VALUE(kc.size(3) == d && vc.sizes() == kc.sizes(),
              "key_cache and value_cache must be (num_blocks, block_size, num_kv_heads, head_dim)");
  CHECK_VALUE(hkv > 0 && hq % hkv == 0, "num_heads must be divisible by num_kv_heads");
  gqa_ragged_args g{};
  g.dtype = dtype16(q);
  g.cache_fp8 = is(kc, at::kFloat8_e4m3fn);
  CHECK_TYPE(vc.scalar_type() == kc.scalar_type() && (g.cache_fp8 || kc.scalar_type() == q.scalar_type()),
             "the caches must share query's dtype, or both be float8_e4m3fn");
  CHECK_TYPE(is(bt, at::kInt) && is(cu, at::kInt) && is(lens, at::kInt), "block_tables, cu_query_lens and seq_lens must be int32");
  CHECK_VALUE(lens.dim() == 1, "seq_lens must be (num_seqs,)");
  const int64_t n = lens.size(0);
  CHECK_VALUE(bt.dim() == 2 && bt.size(0) == n && shaped(cu, {n + 1}),
              "block_tables must be (num_seqs, max_blocks), seq_lens (num_seqs,) and cu_query_lens (num_seqs + 1,)");
  const bool causal = truth(a[9]), window = a[12] != Py_None;
  g.window = window ? integer32(a[12], "window is too large") : 0;
  CHECK_VALUE(!window || g.window >= 1, "window must be at least 1");
  g.softcap = (float)number(a[10]);
  CHECK_VALUE(g.softcap >= 0, "softcap must not be negative");
  CHECK_VALUE(causal || (!window && !prefix.defined()), "window and prefix_lens need causal");
  g.k_scale = (float)number(a[15]);
  g.v_scale = (float)number(a[16]);
  CHECK_VALUE(!g.cache_fp8 || (g.k_scale > 0 && g.v_scale > 0), "fp8 caches need positive k_scale and v_scale");
  CHECK_VALUE(!alibi.defined() || (is(alibi, at::kFloat) && shaped(alibi, {hq})), "alibi_slopes must be float32 (num_heads,)");
  CHECK_VALUE(!prefix.defined() || (is(prefix, at::kInt) && shaped(prefix, {n})), "prefix_lens must be int32 (num_seqs,)");
  CHECK_VALUE(!starts.defined() || (is(starts, at::kInt) && shaped(starts, {tokens})), "key_starts must be int32 (num_tokens,)");
  at::Tensor out = optional(a[18], "out");
  CHECK_VALUE(!out.defined() || (out.sizes() == q.sizes() && out.scalar_type() == q.scalar_type()),
              "out must have query's shape and dtype");
  const int device = device_of({&q, &kc, &vc, &bt, &cu, &lens, &alibi, &prefix, &starts, &out});
  if (!out.defined()) out = empty(q.sizes(), q.scalar_type(), device);
  at::Tensor lse;
  if (truth(a[17])) lse = empty({tokens, hq}, at::kFloat, device);
  q = rows(q);
  bt = flat(bt);
  cu = flat(cu);
  lens = flat(lens);
  alibi = flat(alibi);
  prefix = flat(prefix);
  starts = flat(starts);
  g.q = q.data_ptr();
  g.k_cache = kc.data_ptr();
  g.v_cache = vc.data_ptr();
  g.o = out.data_ptr();
  g.lse = data<float>(lse);
  g.block_table = data<int>(bt);
  g.cu_query_lens = data<int>(cu);
  g.seq_lens = data<int>(lens);
  g.alibi_slopes = data<float>(alibi);
  g.prefix_lens = data<int>(prefix);
  g.key_starts = data<int>(starts);
  strides_of(q, g.q_strides);
  strides_of(kc, g.k_strides);
  strides_of(vc, g.v_strides);
  strides_of(out, g.o_strides);
  g.bt_stride = dim32(bt, 1);
  g.num_seqs = dim32(lens, 0);
  g.num_tokens = dim32(q, 0);
  g.num_heads = dim32(q, 1);
  g.num_kv_heads = dim32(kc, 2);
  g.head_dim = (int)d;
  g.block_size = dim32(kc, 1);
  g.num_blocks = dim32(kc, 0);
  const int64_t capacity = std::min<int64_t>(bt.size(1) * kc.size(1), INT_MAX);
  g.max_query_len = a[6] == Py_None ? g.num_tokens : integer32(a[6], "max_query_len is too large");
  g.max_seq_len = a[7] == Py_None ? (int)capacity : (int)std::min<long long>(integer(a[7]), capacity);
  g.causal = causal;
  g.scale = a[8] == Py_None ? (float)(1.0 / std::sqrt((double)d)) : (float)number(a[8]);
  with_workspace(device, "gqa_ragged_fwd", g, g_lib.ragged, g_lib.ragged_bytes);
  PyObject* r = THPVariable_Wrap(out);
  if (!lse.defined()) return r;
  PyObject* rl = THPVariable_Wrap(lse);
  PyObject* both = PyTuple_Pack(2, r, rl);
  Py_XDECREF(r);
  Py_XDECREF(rl);
  return both;
}

// ----------------------------------------------------------------------------- draft verification
// (draft_tokens, target, draft_probs | None, uniforms | None, exponentials | None, cu, out | None,
//  greedy); the probabilities of the drafts and the random numbers are None if greedy.
// Returns (tokens, num_tokens).
PyObject* verify(PyObject* const* a) {
  at::Tensor d = tensor(a[0], "draft_tokens"), target = tensor(a[1], "the target"), dp = optional(a[2], "draft_probs"),
             u = optional(a[3], "uniforms"), e = optional(a[4], "exponentials"), cu = tensor(a[5], "cu_query_lens");
  const bool greedy = truth(a[7]);
  CHECK_VALUE(d.dim() == 2 && target.dim() == 2, "draft_tokens must be (num_seqs, max_drafts) and the target (num_rows, vocab)");
  const int64_t n = d.size(0), k = d.size(1), vocab = target.size(1);
  gqa_verify_args g{};
  g.dtype = is(target, at::kFloat) ? GQA_DTYPE_F32 : is(target, at::kBFloat16) ? GQA_DTYPE_BF16 : is(target, at::kHalf) ? GQA_DTYPE_F16 : -1;
  CHECK_TYPE(g.dtype >= 0, "float32, bfloat16 or float16 targets are supported");
  CHECK_TYPE(is(d, at::kInt) && is(cu, at::kInt), "draft_tokens and cu_query_lens must be int32");
  CHECK_VALUE(shaped(cu, {n + 1}), "cu_query_lens must be (num_seqs + 1,)");
  CHECK_VALUE(k <= 64, "at most 64 drafted tokens are supported");
  CHECK_VALUE(vocab >= 1, "the target must have a vocabulary");
  if (!greedy) {
    CHECK_VALUE(u.defined() && e.defined() && shaped(u, {n, k}) && shaped(e, {n, vocab}),
                "uniforms must be (num_seqs, max_drafts) and exponentials (num_seqs, vocab)");
    CHECK_TYPE(is(u, at::kFloat) && is(e, at::kFloat), "uniforms and exponentials must be float32");
    if (dp.defined()) {
      CHECK_VALUE(shaped(dp, {n, k, vocab}), "draft_probs must be (num_seqs, max_drafts, vocab)");
      CHECK_TYPE(dp.scalar_type() == target.scalar_type(), "draft_probs must have target_probs' dtype");
    }
  }
  at::Tensor tokens, num;
  if (a[6] != Py_None) {
    CHECK_TYPE(PyTuple_Check(a[6]) && PyTuple_GET_SIZE(a[6]) == 2, "out must be (tokens, num_tokens)");
    tokens = tensor(PyTuple_GET_ITEM(a[6], 0), "out[0]");
    num = tensor(PyTuple_GET_ITEM(a[6], 1), "out[1]");
    CHECK_VALUE(shaped(tokens, {n, k + 1}) && shaped(num, {n}) && is(tokens, at::kInt) && is(num, at::kInt) && tokens.is_contiguous() &&
                    num.is_contiguous(),
                "out must be contiguous int32 (num_seqs, max_drafts + 1) and (num_seqs,)");
  }
  const int device = device_of({&target, &d, &dp, &u, &e, &cu, &tokens, &num});
  if (!tokens.defined()) {
    tokens = empty({n, k + 1}, at::kInt, device);
    num = empty({n}, at::kInt, device);
  }
  auto packed = [](at::Tensor& t) {
    if (t.defined() && !last_dim_ok(t)) t = t.contiguous();
  };
  packed(d);
  packed(target);
  packed(dp);
  packed(u);
  packed(e);
  cu = flat(cu);
  g.draft_tokens = data<int>(d);
  g.target = target.data_ptr();
  g.draft_probs = data<void>(dp);
  g.uniforms = data<float>(u);
  g.exponentials = data<float>(e);
  g.cu_query_lens = data<int>(cu);
  g.tokens = data<int>(tokens);
  g.num_tokens = data<int>(num);
  g.draft_token_stride = d.stride(0);
  g.target_stride = target.stride(0);
  if (dp.defined()) {
    g.draft_strides[0] = dp.stride(0);
    g.draft_strides[1] = dp.stride(1);
  }
  if (!greedy) {
    g.uniform_stride = u.stride(0);
    g.exponential_stride = e.stride(0);
  }
  g.num_seqs = dim32(d, 0);
  g.num_rows = dim32(target, 0);
  g.max_drafts = (int)k;
  g.vocab = dim32(target, 1);
  with_workspace(device, greedy ? "gqa_verify_greedy" : "gqa_verify_drafts", g, greedy ? g_lib.greedy : g_lib.verify,
                 [&](const gqa_verify_args* x) { return g_lib.verify_bytes(x, greedy); });
  PyObject *r0 = THPVariable_Wrap(tokens), *r1 = THPVariable_Wrap(num);
  PyObject* both = PyTuple_Pack(2, r0, r1);
  Py_XDECREF(r0);
  Py_XDECREF(r1);
  return both;
}

// ----------------------------------------------------------------------------- the module
// Runs f with exactly `want` arguments; C++ exceptions become Python's.
template <typename F>
PyObject* guarded(Py_ssize_t got, Py_ssize_t want, F f) {
  if (got != want) {
    PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", want, got);
    return nullptr;
  }
  if (!g_lib.strerror) {
    PyErr_SetString(PyExc_RuntimeError, "the library is not bound");
    return nullptr;
  }
  try {
    return f();
  } catch (const PyError&) {
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
  }
  return nullptr;
}
PyObject* py_step_plan(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 16, [&]() -> PyObject* {
    step_plan(a);
    Py_RETURN_NONE;
  });
}
PyObject* py_norm_rope(PyObject*, PyObject* const* a, Py_ssize_t n) { return guarded(n, 16, [&] { return norm_rope(a); }); }
PyObject* py_ragged(PyObject*, PyObject* const* a, Py_ssize_t n) { return guarded(n, 19, [&] { return ragged(a); }); }
PyObject* py_verify(PyObject*, PyObject* const* a, Py_ssize_t n) { return guarded(n, 8, [&] { return verify(a); }); }
PyObject* py_drop(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 1, [&]() -> PyObject* {
    drop_workspaces((int)integer(a[0]));
    Py_RETURN_NONE;
  });
}
// bind(step_plan, qk_norm_rope, ragged_fwd, ragged_bytes, verify_drafts, verify_greedy, verify_bytes, strerror)
PyObject* py_bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 8) {
    PyErr_SetString(PyExc_TypeError, "bind takes eight addresses");
    return nullptr;
  }
  void* p[8];
  for (int i = 0; i < 8; ++i) {
    p[i] = PyLong_AsVoidPtr(a[i]);
    if (!p[i]) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "null address");
      return nullptr;
    }
  }
  g_lib.step_plan = reinterpret_cast<decltype(g_lib.step_plan)>(p[0]);
  g_lib.rope = reinterpret_cast<decltype(g_lib.rope)>(p[1]);
  g_lib.ragged = reinterpret_cast<decltype(g_lib.ragged)>(p[2]);
  g_lib.ragged_bytes = reinterpret_cast<decltype(g_lib.ragged_bytes)>(p[3]);
  g_lib.verify = reinterpret_cast<decltype(g_lib.verify)>(p[4]);
  g_lib.greedy = reinterpret_cast<decltype(g_lib.greedy)>(p[5]);
  g_lib.verify_bytes = reinterpret_cast<decltype(g_lib.verify_bytes)>(p[6]);
  g_lib.strerror = reinterpret_cast<decltype(g_lib.strerror)>(p[7]);
  Py_RETURN_NONE;
}

#define METHOD(name, f) {name, (PyCFunction)(void (*)(void))f, METH_FASTCALL, nullptr}
PyMethodDef g_methods[] = {METHOD("bind", py_bind),           METHOD("step_plan", py_step_plan), METHOD("norm_rope", py_norm_rope),
                           METHOD("ragged", py_ragged),       METHOD("verify", py_verify),       METHOD("drop_workspaces", py_drop),
                           {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_serving_ext", "Binding of the ragged serving step.", -1, g_methods};

}  // namespace

PyMODINIT_FUNC PyInit__serving_ext(void) { return PyModule_Create(&g_module); }
