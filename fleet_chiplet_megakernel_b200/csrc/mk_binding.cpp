// The serving operators as Python functions: checks of the tensors, outputs and workspaces from torch's allocator, the C entry point on
// the current stream of the tensors' device.  A call of these takes a few microseconds of host time where the same checks in
// Python and ctypes take 30 to 50, several times what the smaller kernels run.
//
// The entry points are those of the library that the package has loaded (bind()); this module is linked with none of it.
#include <ATen/core/Tensor.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/zeros.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>

#include "../../include/b200mk.h"

namespace {

constexpr int64_t kHeadDim = 128;
constexpr int64_t kMaxInt = 0x7fffffff;

struct {
  decltype(&mk_plan_step) plan_step;
  decltype(&mk_rotate_append) rotate_append;
  decltype(&mk_chunk_attention_workspace) attention_workspace;
  decltype(&mk_chunk_attention) attention;
  decltype(&mk_sample_tokens) sample;
  decltype(&mk_op_error) error;
  decltype(&mk_op_check) check;
} g_lib;

// The texts of refusals.
void put(std::string& s, const char* t) { s += t; }
void put(std::string& s, const std::string& t) { s += t; }
void put(std::string& s, int64_t v) { s += std::to_string(v); }
void put(std::string& s, at::IntArrayRef v) {
  s += '[';
  for (size_t i = 0; i < v.size(); ++i) s += (i ? ", " : "") + std::to_string(v[i]);
  s += ']';
}
void put(std::string& s, at::ScalarType t) { s += c10::toString(t); }
void put(std::string& s, const c10::Device& d) { s += d.str(); }
template <typename... P> std::string text(const P&... parts) {
  std::string s;
  (put(s, parts), ...);
  return s;
}
template <typename... P> [[noreturn, gnu::noinline]] void refuse(const P&... parts) { C10_THROW_ERROR(ValueError, text(parts...)); }
template <typename... P> [[noreturn, gnu::noinline]] void too_large(const P&... parts) { C10_THROW_ERROR(NotImplementedError, text(parts...)); }
#define REFUSE_IF(bad, ...) \
  do {                      \
    if (bad) refuse(__VA_ARGS__); \
  } while (0)
#define TOO_LARGE_IF(bad, ...) \
  do {                         \
    if (bad) too_large(__VA_ARGS__); \
  } while (0)
void need(bool ok, const char* what, const char* msg) { REFUSE_IF(!ok, what, msg); }
// A status of the library as the exceptions of PersistentKernel.
void status(int64_t rc) {
  if (rc >= 0) return;
  char said[512] = "";
  g_lib.error(said, sizeof said);
  TOO_LARGE_IF(rc == MK_E_UNSUPPORTED || rc == MK_E_TOO_LARGE, said);
  REFUSE_IF(rc == MK_E_INVALID, said);
  C10_THROW_ERROR(Error, std::string(said));
}

const at::Tensor& tensor(PyObject* o, const char* what) {
  need(THPVariable_Check(o), what, ": a tensor is needed");
  return THPVariable_Unpack(o);
}
const at::Tensor* maybe(PyObject* o, const char* what) { return o == Py_None ? nullptr : &tensor(o, what); }
int64_t number(PyObject* o, const char* what, int64_t lo, int64_t hi) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw python_error();
  REFUSE_IF(v < lo || v > hi, what, ": ", v, ", ", lo, " to ", hi, " is allowed");
  return v;
}
double real(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw python_error();
  return v;
}

struct Checks {
  c10::Device device;
  explicit Checks(const at::Tensor& t, const char* what) : device(t.device()) {
    need(t.is_cuda(), what, " must be a CUDA tensor; there is no CPU fallback");
    plain(t, what);
  }
  static void plain(const at::Tensor& t, const char* what) {
    need(!t.is_neg(), what, " is negated lazily: pass x.resolve_neg()");
    no_gradient(t, what);
  }
  static void no_gradient(const at::Tensor& t, const char* what) {
    need(!t.requires_grad() || !c10::GradMode::is_enabled(), what, " requires a gradient and the serving operators have none: call them under torch.no_grad()");
    need(!t._fw_grad(0).defined(), what, " carries a forward-mode tangent and the serving operators have no derivative: pass torch.autograd.forward_ad.unpack_dual(x).primal");
  }
  void here(const at::Tensor& t, const char* what) const {
    REFUSE_IF(t.device() != device, what, " is on ", t.device(), ", the first tensor on ", device);
    need(t.layout() == at::kStrided, what, ": a strided tensor is needed");
    plain(t, what);
  }
  void type(const at::Tensor& t, const char* what, at::ScalarType dt) const {
    here(t, what);
    REFUSE_IF(t.scalar_type() != dt, what, ".dtype: ", t.scalar_type(), ", ", dt, " is needed");
  }
  // one dimension of n entries (n < 0: of any number), contiguous
  template <typename P = void> P* list(const at::Tensor& t, const char* what, at::ScalarType dt, int64_t n) const {
    type(t, what, dt);
    REFUSE_IF(t.dim() != 1 || (n >= 0 && t.size(0) != n), what, ".shape: ", t.sizes(), ", one dimension", n >= 0 ? " of " + std::to_string(n) : std::string(), " is needed");
    need(t.is_contiguous(), what, " must be contiguous");
    TOO_LARGE_IF(t.size(0) > kMaxInt, what, ": over 2^31 entries");
    return static_cast<P*>(t.data_ptr());
  }
  // [tokens, heads, 128], any token and head stride
  void* rows(const at::Tensor& t, const char* what, at::ScalarType dt, int64_t tokens, int64_t heads, int64_t* stride) const {
    type(t, what, dt);
    REFUSE_IF(t.dim() != 3 || t.size(2) != kHeadDim || (tokens >= 0 && t.size(0) != tokens) || (heads >= 0 && t.size(1) != heads), what, ".shape: ", t.sizes(), ", [", tokens >= 0 ? std::to_string(tokens) : "tokens", ", ", heads >= 0 ? std::to_string(heads) : "heads", ", 128] is needed");
    need(t.stride(2) == 1, what, ": the elements of a row must be contiguous");
    TOO_LARGE_IF(t.size(0) > kMaxInt || t.size(1) > kMaxInt, what, ": over 2^31 rows");
    stride[0] = t.stride(0);
    stride[1] = t.stride(1);
    return t.data_ptr();
  }
  void* cache(const at::Tensor& t, const char* what, at::ScalarType dt, int64_t* stride) const {
    type(t, what, dt);
    REFUSE_IF(t.dim() != 4 || t.size(3) != kHeadDim || t.numel() == 0, what, ".shape: ", t.sizes(), ", [pages, page_size, kv_heads, 128] is needed");
    need(t.stride(3) == 1, what, ": the elements of a row must be contiguous");
    for (int i = 0; i < 3; ++i) {
      TOO_LARGE_IF(t.size(i) > kMaxInt, what, ": over 2^31 pages or rows");
      stride[i] = t.stride(i);
    }
    return t.data_ptr();
  }
  // What is written may not share memory, as the rows of an expanded tensor do: n dimensions of entries of `reach` elements.
  static void apart(const at::Tensor& t, const char* what) { apart(t, what, (int)t.dim() - 1, kHeadDim); }
  static void apart(const at::Tensor& t, const char* what, int n, int64_t reach) {
    bool done[4] = {};
    for (int k = 0; k < n; ++k) {
      int best = -1;
      for (int i = 0; i < n; ++i)
        if (!done[i] && (best < 0 || t.stride(i) < t.stride(best))) best = i;
      done[best] = true;
      if (t.size(best) <= 1) continue;
      need(t.stride(best) >= reach, what, ": its rows share memory");
      reach += t.stride(best) * (t.size(best) - 1);
    }
  }
};
at::ScalarType row_type(const at::Tensor& t, const char* what) {
  REFUSE_IF(t.scalar_type() != at::kBFloat16 && t.scalar_type() != at::kHalf, what, ".dtype: ", t.scalar_type(), ", bf16 or fp16 is needed");
  return t.scalar_type();
}
int code(at::ScalarType t) { return t == at::kBFloat16 ? MK_BF16 : t == at::kHalf ? MK_F16 : MK_F32; }
at::Tensor new_rows(int64_t tokens, int64_t heads, const at::Tensor& like) { return at::zeros({tokens, heads, kHeadDim}, like.options().requires_grad(false)); }
void count(Py_ssize_t n, Py_ssize_t want) { TORCH_CHECK(n == want, n, " arguments, ", want, " are needed"); }

PyObject* bind(PyObject*, PyObject* const* v, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 7);
  auto at = [&](int i) { return PyLong_AsVoidPtr(v[i]); };
  g_lib.plan_step = reinterpret_cast<decltype(g_lib.plan_step)>(at(0));
  g_lib.rotate_append = reinterpret_cast<decltype(g_lib.rotate_append)>(at(1));
  g_lib.attention_workspace = reinterpret_cast<decltype(g_lib.attention_workspace)>(at(2));
  g_lib.attention = reinterpret_cast<decltype(g_lib.attention)>(at(3));
  g_lib.sample = reinterpret_cast<decltype(g_lib.sample)>(at(4));
  g_lib.error = reinterpret_cast<decltype(g_lib.error)>(at(5));
  g_lib.check = reinterpret_cast<decltype(g_lib.check)>(at(6));
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

PyObject* check_waits(PyObject*, PyObject* const*, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 0);
  status(g_lib.check());
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

PyObject* plan_step(PyObject*, PyObject* const* v, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 14);
  mk_step_plan_args a = {};
  const at::Tensor& lengths = tensor(v[0], "lengths");
  const Checks c(lengths, "lengths");
  a.lengths = c.list<int32_t>(lengths, "lengths", at::kInt, -1);
  const int64_t R = lengths.size(0);
  need(R > 0, "lengths", ": a length per request is needed");
  a.new_tokens = c.list<int32_t>(tensor(v[1], "new_tokens"), "new_tokens", at::kInt, R);
  const at::Tensor& table = tensor(v[2], "block_table");
  c.type(table, "block_table", at::kInt);
  REFUSE_IF(table.dim() != 2 || table.size(0) != R || table.size(1) < 1 || table.size(1) > kMaxInt, "block_table.shape: ", table.sizes(), ", [", R, ", pages of the longest request] is needed");
  need(table.stride(1) == 1 && (R == 1 || table.stride(0) >= table.size(1)), "block_table", ": rows must be contiguous and apart");
  a.block_table = static_cast<int32_t*>(table.data_ptr());
  a.table_width = (int32_t)table.size(1);
  a.table_stride = R == 1 ? table.size(1) : table.stride(0);
  const at::Tensor& ring = tensor(v[3], "free_pages");
  a.free_pages = c.list<int32_t>(ring, "free_pages", at::kInt, -1);
  a.free_range_in = c.list<int64_t>(tensor(v[4], "free_range"), "free_range", at::kLong, 2);
  a.page_size = (int32_t)number(v[5], "page_size", 1, kMaxInt);
  a.qo_indptr = c.list<int32_t>(tensor(v[6], "plan.qo_indptr"), "plan.qo_indptr", at::kInt, R + 1);
  a.kv_indptr = c.list<int32_t>(tensor(v[7], "plan.kv_indptr"), "plan.kv_indptr", at::kInt, R + 1);
  const at::Tensor& indices = tensor(v[8], "plan.kv_indices");
  a.kv_indices = c.list<int32_t>(indices, "plan.kv_indices", at::kInt, -1);
  a.last_page_len = c.list<int32_t>(tensor(v[9], "plan.last_page_len"), "plan.last_page_len", at::kInt, R);
  const at::Tensor& slots = tensor(v[10], "plan.slots");
  a.slots = c.list<int64_t>(slots, "plan.slots", at::kLong, -1);
  a.positions = c.list<int32_t>(tensor(v[11], "plan.positions"), "plan.positions", at::kInt, slots.size(0));
  a.granted = c.list<int32_t>(tensor(v[12], "plan.granted"), "plan.granted", at::kInt, R);
  a.free_range_out = c.list<int64_t>(tensor(v[13], "plan.free_range"), "plan.free_range", at::kLong, 2);
  need(a.free_range_out != a.free_range_in, "plan.free_range", " may not be free_range: the call reads one and writes the other");
  a.requests = (int32_t)std::min(R, kMaxInt);
  a.ring_size = (int32_t)ring.size(0);
  a.max_indices = (int32_t)indices.size(0);
  a.max_tokens = (int32_t)slots.size(0);
  const c10::cuda::CUDAGuard guard(c.device);
  status(g_lib.plan_step(&a, at::cuda::getCurrentCUDAStream().stream()));
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

PyObject* rotate_append(PyObject*, PyObject* const* v, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 13);
  mk_rotate_append_args a = {};
  const at::Tensor& q = tensor(v[0], "q");
  const Checks c(q, "q");
  const at::ScalarType dt = row_type(q, "q");
  a.q = c.rows(q, "q", dt, -1, -1, a.q_stride);
  const at::Tensor& k = tensor(v[1], "k");
  const int64_t T = q.size(0), n_q = q.size(1);
  a.k = c.rows(k, "k", dt, T, -1, a.k_stride);
  const int64_t n_kv = k.size(1);
  a.v = c.rows(tensor(v[2], "v"), "v", dt, T, n_kv, a.v_stride);
  const at::Tensor &cos = tensor(v[3], "cos"), &sin = tensor(v[4], "sin");
  for (const at::Tensor* t : {&cos, &sin}) {
    const char* what = t == &cos ? "cos" : "sin";
    c.here(*t, what);
    REFUSE_IF(t->dim() != 2 || t->size(1) != kHeadDim || t->size(0) < 1 || t->size(0) > kMaxInt || t->stride(1) != 1 || t->sizes() != cos.sizes(), what, ".shape: ", t->sizes(), ", [positions, 128] with contiguous rows, cos and sin alike, is needed");
    REFUSE_IF((t->scalar_type() != dt && t->scalar_type() != at::kFloat) || t->scalar_type() != cos.scalar_type(), what, ".dtype: ", t->scalar_type(), ", ", dt, " or fp32, cos and sin alike, is needed");
  }
  a.cos = cos.data_ptr();
  a.sin = sin.data_ptr();
  a.table_stride[0] = cos.stride(0);
  a.table_stride[1] = sin.stride(0);
  a.positions = c.list<int32_t>(tensor(v[5], "positions"), "positions", at::kInt, T);
  a.slots = c.list<int64_t>(tensor(v[6], "slots"), "slots", at::kLong, T);
  const at::Tensor &kc = tensor(v[7], "k_cache"), &vc = tensor(v[8], "v_cache");
  a.k_cache = c.cache(kc, "k_cache", dt, a.k_cache_stride);
  a.v_cache = c.cache(vc, "v_cache", dt, a.v_cache_stride);
  REFUSE_IF(kc.size(2) != n_kv || vc.sizes() != kc.sizes(), "caches of shape ", kc.sizes(), " and ", vc.sizes(), " for ", n_kv, " kv heads");
  Checks::apart(kc, "k_cache");
  Checks::apart(vc, "v_cache");
  if (const at::Tensor* t = maybe(v[9], "q_norm")) a.q_norm = c.list(*t, "q_norm", dt, kHeadDim);
  if (const at::Tensor* t = maybe(v[10], "k_norm")) a.k_norm = c.list(*t, "k_norm", dt, kHeadDim);
  a.eps = (float)real(v[11]);
  const c10::cuda::CUDAGuard guard(c.device);
  at::Tensor out = v[12] == Py_None ? new_rows(T, n_q, q) : tensor(v[12], "out");
  a.out = c.rows(out, "out", dt, T, n_q, a.out_stride);
  Checks::apart(out, "out");
  need(a.out != a.q || (a.out_stride[0] == a.q_stride[0] && a.out_stride[1] == a.q_stride[1]), "out", " shares memory with q and has other strides");
  a.dtype = code(dt);
  a.table_dtype = code(cos.scalar_type());
  a.tokens = (int32_t)T;
  a.q_heads = (int32_t)n_q;
  a.kv_heads = (int32_t)n_kv;
  a.pages = (int32_t)kc.size(0);
  a.page_size = (int32_t)kc.size(1);
  a.table_rows = (int32_t)cos.size(0);
  if (T > 0) status(g_lib.rotate_append(&a, at::cuda::getCurrentCUDAStream().stream()));
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

PyObject* chunk_attention(PyObject*, PyObject* const* v, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 13);
  mk_chunk_attention_args a = {};
  const at::Tensor& q = tensor(v[0], "q");
  const Checks c(q, "q");
  const at::ScalarType dt = row_type(q, "q");
  a.q = c.rows(q, "q", dt, -1, -1, a.q_stride);
  const int64_t T = q.size(0), n_q = q.size(1);
  const at::Tensor &kc = tensor(v[1], "k_cache"), &vc = tensor(v[2], "v_cache");
  a.k_cache = c.cache(kc, "k_cache", dt, a.k_cache_stride);
  a.v_cache = c.cache(vc, "v_cache", dt, a.v_cache_stride);
  REFUSE_IF(vc.sizes() != kc.sizes(), "k_cache is ", kc.sizes(), ", v_cache ", vc.sizes());
  const int64_t n_kv = kc.size(2);
  REFUSE_IF(n_q % n_kv, n_q, " q heads on ", n_kv, " kv heads");
  const at::Tensor& last = tensor(v[6], "last_page_len");
  a.last_page_len = c.list<int32_t>(last, "last_page_len", at::kInt, -1);
  const int64_t R = last.size(0);
  a.qo_indptr = c.list<int32_t>(tensor(v[3], "qo_indptr"), "qo_indptr", at::kInt, R + 1);
  a.kv_indptr = c.list<int32_t>(tensor(v[4], "kv_indptr"), "kv_indptr", at::kInt, R + 1);
  const at::Tensor& indices = tensor(v[5], "kv_indices");
  a.kv_indices = c.list<int32_t>(indices, "kv_indices", at::kInt, -1);
  a.scale = v[7] == Py_None ? (float)(1.0 / std::sqrt((double)kHeadDim)) : (float)real(v[7]);
  a.window = (int32_t)number(v[8], "window", 0, kMaxInt);
  a.sinks = (int32_t)number(v[9], "sinks", 0, kMaxInt);
  const c10::cuda::CUDAGuard guard(c.device);
  at::Tensor out = v[10] == Py_None ? new_rows(T, n_q, q) : tensor(v[10], "out");
  a.out = c.rows(out, "out", dt, T, n_q, a.out_stride);
  Checks::apart(out, "out");
  need(a.out != a.q || T * n_q == 0, "out", " may not be q");
  if (const at::Tensor* t = maybe(v[11], "lse")) {
    c.type(*t, "lse", at::kFloat);
    REFUSE_IF(t->dim() != 2 || t->size(0) != T || t->size(1) != n_q, "lse.shape: ", t->sizes(), ", [", T, ", ", n_q, "] is needed");
    Checks::apart(*t, "lse", 2, 1);
    a.lse = static_cast<float*>(t->data_ptr());
    a.lse_stride[0] = t->stride(0);
    a.lse_stride[1] = t->stride(1);
  }
  a.max_new = (int32_t)number(v[12], "max_new", 0, kMaxInt);
  a.dtype = code(dt);
  a.requests = (int32_t)R;
  a.tokens = (int32_t)T;
  a.q_heads = (int32_t)n_q;
  a.kv_heads = (int32_t)n_kv;
  a.page_size = (int32_t)kc.size(1);
  a.pages = (int32_t)kc.size(0);
  a.num_indices = (int32_t)indices.size(0);
  if (T > 0 && R > 0 && n_q > 0) {
    a.workspace_bytes = g_lib.attention_workspace(&a);
    status(a.workspace_bytes);
    // of the current stream's pool, or of the graph that captures the call
    const at::Tensor workspace = at::empty({a.workspace_bytes}, q.options().dtype(at::kByte).requires_grad(false));
    a.workspace = workspace.data_ptr();
    status(g_lib.attention(&a, at::cuda::getCurrentCUDAStream().stream()));
  }
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

PyObject* sample_tokens(PyObject*, PyObject* const* v, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 9);
  mk_sample_args a = {};
  const at::Tensor& logits = tensor(v[0], "logits");
  const Checks c(logits, "logits");
  const at::ScalarType dt = logits.scalar_type();
  REFUSE_IF(dt != at::kBFloat16 && dt != at::kHalf && dt != at::kFloat, "logits.dtype: ", dt, ", bf16, fp16 or fp32 is needed");
  REFUSE_IF(logits.dim() != 2 || logits.size(1) < 1 || logits.size(1) > kMaxInt || logits.size(0) > kMaxInt, "logits.shape: ", logits.sizes(), ", [rows, vocab] is needed");
  need(logits.stride(1) == 1 || logits.size(1) == 1, "logits", ": the elements of a row must be contiguous");
  const at::Tensor& u = tensor(v[1], "u");
  a.u = c.list<float>(u, "u", at::kFloat, -1);
  const int64_t R = u.size(0);
  if (THPVariable_Check(v[2])) a.temperature = c.list<float>(tensor(v[2], "temperature"), "temperature", at::kFloat, R);
  else a.temperature_value = (float)real(v[2]);
  if (THPVariable_Check(v[3])) a.top_k = c.list<int32_t>(tensor(v[3], "top_k"), "top_k", at::kInt, R);
  else a.top_k_value = (int32_t)number(v[3], "top_k", -kMaxInt, kMaxInt);
  if (THPVariable_Check(v[4])) a.top_p = c.list<float>(tensor(v[4], "top_p"), "top_p", at::kFloat, R);
  else a.top_p_value = (float)real(v[4]);
  if (THPVariable_Check(v[5])) a.min_p = c.list<float>(tensor(v[5], "min_p"), "min_p", at::kFloat, R);
  else a.min_p_value = (float)real(v[5]);
  if (const at::Tensor* t = maybe(v[6], "qo_indptr")) a.qo_indptr = c.list<int32_t>(*t, "qo_indptr", at::kInt, R + 1);
  else REFUSE_IF(logits.size(0) < R, logits.size(0), " rows of logits for ", R, " requests");
  const c10::cuda::CUDAGuard guard(c.device);
  at::Tensor out = v[7] == Py_None ? at::empty({R}, logits.options().dtype(at::kLong).requires_grad(false)) : tensor(v[7], "out");
  a.tokens = c.list<int64_t>(out, "out", at::kLong, R);
  const int asked = PyObject_IsTrue(v[8]);
  if (asked < 0) throw python_error();
  const bool with_logprobs = asked != 0;
  at::Tensor logprobs;
  if (with_logprobs) {
    logprobs = at::empty({R}, logits.options().dtype(at::kFloat).requires_grad(false));
    a.logprobs = static_cast<float*>(logprobs.data_ptr());
  }
  a.logits = logits.data_ptr();
  a.row_stride = logits.stride(0);
  a.dtype = code(dt);
  a.requests = (int32_t)R;
  a.rows = (int32_t)logits.size(0);
  a.vocab = (int32_t)logits.size(1);
  if (R > 0) status(g_lib.sample(&a, at::cuda::getCurrentCUDAStream().stream()));
  if (!with_logprobs) return THPVariable_Wrap(std::move(out));
  PyObject* pair = PyTuple_New(2);
  if (!pair) throw python_error();
  PyTuple_SET_ITEM(pair, 0, THPVariable_Wrap(std::move(out)));
  PyTuple_SET_ITEM(pair, 1, THPVariable_Wrap(std::move(logprobs)));
  return pair;
  END_HANDLE_TH_ERRORS
}

#define MK_METHOD(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(f)), METH_FASTCALL, nullptr}
PyMethodDef g_methods[] = {MK_METHOD(bind), MK_METHOD(check_waits), MK_METHOD(plan_step), MK_METHOD(rotate_append), MK_METHOD(chunk_attention), MK_METHOD(sample_tokens), {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_serving_native", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__serving_native() { return PyModule_Create(&g_module); }
