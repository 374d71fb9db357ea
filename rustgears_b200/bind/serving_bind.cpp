// serving_bind.cpp -- Python binding of the decoder-serving entry points (include/rg_npu.h) on
// torch tensors: checks of shapes, dtypes, strides and devices, the outputs' allocation, the
// call on the tensors' device and its current stream.
//
// A decode step is a chain of calls of a few microseconds of device time each, so the host side
// of a call counts: through ctypes and torch's Python attributes one took 8 to 15 us, here 3 to 5.
// rustgears_b200/serving.py documents the functions and is the interface; it passes every
// argument by position.
#include <Python.h>
#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/Dtype.h>

#include <cmath>
#include <sstream>
#include <stdexcept>

#include "rg_npu.h"

namespace {

PyObject* g_check = nullptr;  // rustgears_b200._native.check: raises a status as RgError

// ---------------------------------------------------------------------------
// refusals (ValueError)
// ---------------------------------------------------------------------------
template <typename... A>
[[noreturn]] void refuse(const A&... parts) {
  std::ostringstream s;
  (s << ... << parts);
  throw std::invalid_argument(s.str());
}

struct Raised {};  // a Python exception is set

// ---------------------------------------------------------------------------
// arguments
// ---------------------------------------------------------------------------
const at::Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) refuse(name, ": a tensor is needed");
  return THPVariable_Unpack(o);
}
const at::Tensor* optional(PyObject* o, const char* name) {
  return o == Py_None ? nullptr : &tensor(o, name);
}
long long integer(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw Raised{};
  return v;
}
bool truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw Raised{};
  return v != 0;
}
int32_t int32(PyObject* o, const char* name) {
  const long long v = integer(o);
  if (v < INT32_MIN || v > INT32_MAX) refuse(name, ": ", v, " is no 32-bit integer");
  return (int32_t)v;
}

int32_t dtype_code(at::ScalarType t) {
  return t == at::kFloat ? RG_DTYPE_F32 : t == at::kHalf ? RG_DTYPE_F16 : t == at::kBFloat16 ? RG_DTYPE_BF16 : -1;
}
int32_t need_dtype(at::ScalarType t, const char* name) {
  const int32_t c = dtype_code(t);
  if (c < 0) refuse(name, ": float32, float16 or bfloat16 is needed, got ", c10::toString(t));
  return c;
}

// The common CUDA device of the tensors.
struct Device {
  int index = -1;
  void first(const at::Tensor& t) {
    if (!t.is_cuda()) throw std::invalid_argument("serving operators need CUDA tensors");
    index = t.get_device();
  }
  void also(const at::Tensor& t) const {
    if (!t.is_cuda() || t.get_device() != index)
      refuse("tensors on cuda:", index, " and ", t.device().str());
  }
  void also(const at::Tensor* t) const {
    if (t) also(*t);
  }
};

at::Tensor empty(at::IntArrayRef shape, at::ScalarType t, int device) {
  return at::detail::empty_cuda(shape, t, c10::Device(c10::kCUDA, (c10::DeviceIndex)device), std::nullopt);
}

// A device's two error words, zeroed by its first call and kept for the process.
constexpr int kDevices = 64;
at::Tensor g_words[kDevices];

int32_t* error_words(int device) {
  if (device >= kDevices) refuse("cuda:", device);
  at::Tensor& w = g_words[device];
  if (!w.defined()) {
    const auto st = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device);
    cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
    if (cudaStreamIsCapturing(st.stream(), &cap) != cudaSuccess || cap != cudaStreamCaptureStatusNone)
      throw std::runtime_error("call a serving operator once on this device before capturing a graph");
    at::Tensor z = at::zeros({2}, at::TensorOptions().dtype(at::kInt).device(at::kCUDA, device));
    st.synchronize();  // zeroed before any stream's kernel sets it
    w = z;
  }
  return w.data_ptr<int32_t>();
}

void raise(rg_status st) {
  PyObject* r = PyObject_CallFunction(g_check, "i", (int)st);
  Py_XDECREF(r);
  if (r) throw std::runtime_error("status without an exception");
  throw Raised{};
}

// f(stream) with `device` current, on its current stream.
template <typename F>
void call(int device, F f) {
  c10::cuda::CUDAGuard guard((c10::DeviceIndex)device);
  void* stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream();
  rg_status st;
  Py_BEGIN_ALLOW_THREADS;
  st = f(stream);
  Py_END_ALLOW_THREADS;
  if (st != RG_OK) raise(st);
}

// [tokens, heads, head_dim] with head_dim contiguous; the strides of a dimension of one (torch
// leaves them arbitrary) are 0.
struct Heads {
  int64_t n, h, d, ts, hs;
  Heads(const at::Tensor& t, const char* name, bool written = false) {
    if (t.dim() != 3 || t.stride(2) != 1)
      refuse(name, ": [tokens, heads, head_dim] with contiguous head_dim is needed, got shape ", t.sizes(),
             ", strides ", t.strides());
    n = t.size(0);
    h = t.size(1);
    d = t.size(2);
    ts = n == 1 ? 0 : t.stride(0);
    hs = h == 1 ? 0 : t.stride(1);
    if (written && ((n > 1 && ts == 0) || (h > 1 && hs == 0)))
      refuse(name, ": an expanded tensor cannot be written");
    if (h > INT32_MAX || d > INT32_MAX) refuse(name, ": too large");
  }
};

void vector(const at::Tensor& t, const char* name, at::ScalarType type, int64_t n) {
  if (t.scalar_type() != type || t.dim() != 1 || t.size(0) != n || !t.is_contiguous())
    refuse(name, ": a contiguous ", c10::toString(type), " vector of ", n, " is needed, got ",
           c10::toString(t.scalar_type()), " ", t.sizes());
}

void rotation(const at::Tensor& table, int64_t head_dim) {
  if (table.dim() != 2 || table.scalar_type() != at::kFloat || !table.is_contiguous())
    refuse("table: contiguous float32 [positions, rot_dim] is needed");
  if (table.size(1) > head_dim) refuse("table: rot_dim ", table.size(1), " exceeds head_dim ", head_dim);
}

rg_kv_cache cache_of(const at::Tensor& k, const at::Tensor& v) {
  if (k.dim() != 4 || k.sizes() != v.sizes() || k.scalar_type() != v.scalar_type() || k.stride(3) != 1 ||
      v.stride(3) != 1)
    refuse("caches: two [pages, page_size, kv_heads, head_dim] tensors of one dtype with contiguous head_dim are "
           "needed");
  const at::ScalarType t = k.scalar_type();
  if (t != at::kHalf && t != at::kBFloat16) refuse("caches: float16 or bfloat16 is needed, got ", c10::toString(t));
  int64_t s[3];
  for (int i = 0; i < 3; ++i) {
    s[i] = k.size(i) > 1 ? k.stride(i) : 0;
    if (k.size(i) > 1 && k.stride(i) != v.stride(i)) refuse("caches: the key and value tensors have different strides");
    if (k.size(i) > 1 && s[i] == 0) refuse("caches: an expanded tensor cannot be a cache");
    if (k.size(i) > INT32_MAX) refuse("caches: too large");
  }
  rg_kv_cache c;
  c.k = k.data_ptr();
  c.v = v.data_ptr();
  c.dtype = dtype_code(t);
  c.pages = k.size(0);
  c.page_size = (int32_t)k.size(1);
  c.kv_heads = (int32_t)k.size(2);
  c.head_dim = (int32_t)k.size(3);
  c.page_stride = s[0];
  c.token_stride = s[1];
  c.head_stride = s[2];
  return c;
}

// x [..., k] as rows [m, k] with contiguous rows that do not overlap (a copy only if it has to be)
at::Tensor rows_of(const at::Tensor& x) {
  need_dtype(x.scalar_type(), "x");
  if (x.dim() < 1 || x.size(-1) == 0) refuse("x: [..., k] with k > 0 is needed, got ", x.sizes());
  at::Tensor r = x.dim() == 2 ? x : x.reshape({-1, x.size(-1)});
  const int64_t m = r.size(0), k = r.size(1);
  if ((k > 1 && r.stride(1) != 1) || (m > 1 && r.stride(0) < k)) r = r.contiguous();
  return r;
}
int64_t ldx_of(const at::Tensor& r) { return r.size(0) > 1 ? r.stride(0) : r.size(1); }
// Whether rows_of's rows and a contiguous tensor lie in overlapping ranges of memory.
bool ranges_meet(const at::Tensor& r, const at::Tensor& out) {
  const char *x = static_cast<const char*>(r.data_ptr()), *o = static_cast<const char*>(out.data_ptr());
  const int64_t size = ((r.size(0) - 1) * ldx_of(r) + r.size(1)) * (int64_t)r.element_size();
  return x < o + out.nbytes() && o < x + size;
}

// ---------------------------------------------------------------------------
// the calls
// ---------------------------------------------------------------------------
// x
PyObject* quantize(PyObject* const* o) {
  const at::Tensor x = rows_of(tensor(o[0], "x"));
  Device dev;
  dev.first(x);
  const int64_t m = x.size(0), k = x.size(1), ld = (k + 15) / 16 * 16;
  at::Tensor q = empty({m, ld}, at::kChar, dev.index), s = empty({m}, at::kFloat, dev.index);
  call(dev.index, [&](void* st) {
    return rg_quantize_token_i8(x.data_ptr(), dtype_code(x.scalar_type()), m, k, ldx_of(x), q.data_ptr<int8_t>(), ld,
                                s.data_ptr<float>(), st);
  });
  PyObject* a = THPVariable_Wrap(q);
  PyObject* b = THPVariable_Wrap(s);
  PyObject* both = PyTuple_Pack(2, a, b);
  Py_DECREF(a);
  Py_DECREF(b);
  return both;
}

// x, w, w_scale, bias, act code, act parameter, out dtype, out
PyObject* linear(PyObject* const* o) {
  const at::Tensor& x = tensor(o[0], "x");
  const at::Tensor r = rows_of(x);
  const at::Tensor &w = tensor(o[1], "w"), &ws = tensor(o[2], "w_scale");
  const at::Tensor *bias = optional(o[3], "bias"), *given = optional(o[7], "out");
  const int64_t m = r.size(0), k = r.size(1);
  if (w.dim() != 2 || w.scalar_type() != at::kChar || !w.is_contiguous() || w.size(1) < k || w.size(1) % 16)
    refuse("w: contiguous int8 [n, ld] with ld >= ", k, ", a multiple of 16, is needed, got ",
           c10::toString(w.scalar_type()), " ", w.sizes());
  const int64_t n = w.size(0), ld = w.size(1);
  vector(ws, "w_scale", at::kFloat, n);
  if (bias) vector(*bias, "bias", at::kFloat, n);
  at::ScalarType type = x.scalar_type();
  if (o[6] != Py_None) {
    if (!THPDtype_Check(o[6])) refuse("out_dtype: a torch dtype is needed");
    type = reinterpret_cast<THPDtype*>(o[6])->scalar_type;
  }
  const int32_t code = need_dtype(type, "out_dtype");
  rg_linear_token_args a;
  a.act = int32(o[4], "act");
  a.act_param = (float)PyFloat_AsDouble(o[5]);
  if (PyErr_Occurred()) throw Raised{};
  c10::SmallVector<int64_t, 6> shape(x.sizes().begin(), x.sizes().end());
  shape.back() = n;
  if (given && (given->scalar_type() != type || given->sizes() != at::IntArrayRef(shape) || !given->is_contiguous()))
    refuse("out: contiguous ", c10::toString(type), " ", at::IntArrayRef(shape), " is needed, got ",
           c10::toString(given->scalar_type()), " ", given->sizes());
  Device dev;
  dev.first(r);
  dev.also(w);
  dev.also(ws);
  dev.also(bias);
  dev.also(given);
  at::Tensor out = given ? *given : empty(shape, type, dev.index);
  if (m > 0) {
    const int64_t need = rg_linear_i8_token_workspace_size(m, n, ld);
    if (need == 0 && given && ranges_meet(r, out)) {
      // one launch would write out while it reads x: quantized first, as larger calls do
      at::Tensor q = empty({m, ld}, at::kChar, dev.index), s = empty({m}, at::kFloat, dev.index);
      int32_t* words = error_words(dev.index);
      call(dev.index, [&](void* st) {
        const rg_status e = rg_quantize_token_i8(r.data_ptr(), dtype_code(r.scalar_type()), m, k, ldx_of(r),
                                                 q.data_ptr<int8_t>(), ld, s.data_ptr<float>(), st);
        if (e != RG_OK) return e;
        return rg_gemm_i8_token(q.data_ptr<int8_t>(), s.data_ptr<float>(), w.data_ptr<int8_t>(), ws.data_ptr<float>(),
                                m, n, ld, bias ? bias->data_ptr<float>() : nullptr, a.act, a.act_param, out.data_ptr(),
                                code, n, words, st);
      });
      return THPVariable_Wrap(out);
    }
    at::Tensor space;
    if (need > 0) space = empty({need}, at::kByte, dev.index);
    a.x = r.data_ptr();
    a.w = w.data_ptr<int8_t>();
    a.w_scale = ws.data_ptr<float>();
    a.bias = bias ? bias->data_ptr<float>() : nullptr;
    a.out = out.data_ptr();
    a.m = m; a.k = k; a.ldx = ldx_of(r); a.n = n; a.ld = ld; a.ldo = n;
    a.x_dtype = dtype_code(r.scalar_type());
    a.out_dtype = code;
    int32_t* words = error_words(dev.index);
    call(dev.index, [&](void* st) { return rg_linear_i8_token(&a, need > 0 ? space.data_ptr() : nullptr, words, st); });
  }
  return THPVariable_Wrap(out);
}

// x, positions, table, interleaved, out
PyObject* rope(PyObject* const* o) {
  const at::Tensor &x = tensor(o[0], "x"), &pos = tensor(o[1], "positions"), &table = tensor(o[2], "table");
  const at::Tensor* given = optional(o[4], "out");
  const Heads hx(x, "x");
  const int32_t dt = need_dtype(x.scalar_type(), "x");
  vector(pos, "positions", at::kInt, hx.n);
  rotation(table, hx.d);
  if (given && (given->scalar_type() != x.scalar_type() || given->sizes() != x.sizes()))
    refuse("out: x's shape and dtype are needed");
  if (given) Heads(*given, "out", true);
  Device dev;
  dev.first(x);
  dev.also(pos);
  dev.also(table);
  dev.also(given);
  at::Tensor out = given ? *given : empty(x.sizes(), x.scalar_type(), dev.index);
  if (hx.n > 0 && hx.h > 0) {
    const Heads ho(out, "out", true);
    rg_rope_args a;
    a.x = x.data_ptr();
    a.out = out.data_ptr();
    a.token_stride = hx.ts; a.head_stride = hx.hs; a.out_token_stride = ho.ts; a.out_head_stride = ho.hs;
    a.positions = pos.data_ptr<int32_t>();
    a.table = table.data_ptr<float>();
    a.table_rows = table.size(0);
    a.tokens = hx.n;
    a.dtype = dt;
    a.heads = (int32_t)hx.h; a.head_dim = (int32_t)hx.d; a.rot_dim = (int32_t)table.size(1);
    a.interleaved = truth(o[3]);
    int32_t* words = error_words(dev.index);
    call(dev.index, [&](void* st) { return rg_rope(&a, words, st); });
  }
  return THPVariable_Wrap(out);
}

// k, v, k_cache, v_cache, slots, positions, table, interleaved, q, q_out
PyObject* append(PyObject* const* o) {
  const at::Tensor &k = tensor(o[0], "k"), &v = tensor(o[1], "v"), &kc = tensor(o[2], "k_cache"),
                   &vc = tensor(o[3], "v_cache"), &slots = tensor(o[4], "slots");
  const at::Tensor *pos = optional(o[5], "positions"), *table = optional(o[6], "table"), *q = optional(o[8], "q"),
                   *given = optional(o[9], "q_out");
  const Heads hk(k, "k"), hv(v, "v");
  const rg_kv_cache c = cache_of(kc, vc);
  if (k.sizes() != v.sizes() || hk.h != c.kv_heads || hk.d != c.head_dim)
    refuse("k ", k.sizes(), ", v ", v.sizes(), " do not fit ", kc.sizes());
  const at::ScalarType dt = k.scalar_type(), ct = kc.scalar_type();
  if ((dt != at::kFloat && dt != ct) || v.scalar_type() != dt)
    refuse("k and v: float32 or ", c10::toString(ct), " is needed, got ", c10::toString(dt), " and ",
           c10::toString(v.scalar_type()));
  vector(slots, "slots", at::kLong, hk.n);
  rg_kv_append_args a = {};
  if (table) {
    if (!pos) refuse("positions are needed with a table");
    vector(*pos, "positions", at::kInt, hk.n);
    rotation(*table, hk.d);
  }
  if (given && !q) refuse("q_out without q");
  Device dev;
  dev.first(k);
  dev.also(v);
  dev.also(kc);
  dev.also(vc);
  dev.also(slots);
  dev.also(pos);
  dev.also(table);
  dev.also(q);
  dev.also(given);
  at::Tensor q_out;
  if (q) {
    const Heads hq(*q, "q");
    if (q->scalar_type() != dt || hq.n != hk.n || hq.d != hk.d || hq.h == 0)
      refuse("q: ", c10::toString(dt), " [", hk.n, ", heads, ", hk.d, "] is needed, got ",
             c10::toString(q->scalar_type()), " ", q->sizes());
    if (given && (given->scalar_type() != ct || given->sizes() != q->sizes()))
      refuse("q_out: ", c10::toString(ct), " of q's shape is needed");
    q_out = given ? *given : empty(q->sizes(), ct, dev.index);
    const Heads ho(q_out, "q_out", true);
    a.q = q->data_ptr();
    a.q_out = q_out.data_ptr();
    a.heads = (int32_t)hq.h;
    a.q_token_stride = hq.ts; a.q_head_stride = hq.hs; a.q_out_token_stride = ho.ts; a.q_out_head_stride = ho.hs;
  }
  if (hk.n > 0) {
    a.k = k.data_ptr();
    a.v = v.data_ptr();
    a.k_token_stride = hk.ts; a.k_head_stride = hk.hs; a.v_token_stride = hv.ts; a.v_head_stride = hv.hs;
    a.slots = slots.data_ptr<int64_t>();
    if (table) {
      a.positions = pos->data_ptr<int32_t>();
      a.table = table->data_ptr<float>();
      a.table_rows = table->size(0);
      a.rot_dim = (int32_t)table->size(1);
    }
    a.tokens = hk.n;
    a.x_dtype = dtype_code(dt);
    a.interleaved = truth(o[7]);
    int32_t* words = error_words(dev.index);
    call(dev.index, [&](void* st) { return rg_kv_append(&c, &a, words, st); });
  }
  if (!q) Py_RETURN_NONE;
  return THPVariable_Wrap(q_out);
}

// q, k_cache, v_cache, block_table, kv_len, cu_q, max_q_len, max_kv_len, scale, causal, out
PyObject* attention(PyObject* const* o) {
  const at::Tensor &q = tensor(o[0], "q"), &kc = tensor(o[1], "k_cache"), &vc = tensor(o[2], "v_cache"),
                   &bt = tensor(o[3], "block_table"), &kl = tensor(o[4], "kv_len"), &cu = tensor(o[5], "cu_q");
  const at::Tensor* given = optional(o[10], "out");
  const Heads hq(q, "q");
  const rg_kv_cache c = cache_of(kc, vc);
  if (q.scalar_type() != kc.scalar_type() || hq.d != c.head_dim || hq.h == 0 || c.kv_heads == 0 || hq.h % c.kv_heads)
    refuse("q ", c10::toString(q.scalar_type()), " ", q.sizes(), " does not fit ", c10::toString(kc.scalar_type()), " ",
           kc.sizes());
  const int64_t batch = kl.numel();
  vector(kl, "kv_len", at::kInt, batch);
  vector(cu, "cu_q", at::kInt, batch + 1);
  if (bt.scalar_type() != at::kInt || bt.dim() != 2 || bt.size(0) != batch || (bt.size(1) > 1 && bt.stride(1) != 1))
    refuse("block_table: int32 [", batch, ", max_pages] with contiguous rows is needed");
  if (given && (given->scalar_type() != q.scalar_type() || given->sizes() != q.sizes()))
    refuse("out: q's shape and dtype are needed");
  rg_paged_attention_args a;
  if (batch > INT32_MAX || bt.size(1) > INT32_MAX) refuse("block_table: too large");
  a.batch = (int32_t)batch;
  a.max_pages = (int32_t)bt.size(1);
  a.max_q_len = int32(o[6], "max_q_len");
  if (o[7] == Py_None) {
    const int64_t room = (int64_t)a.max_pages * c.page_size;
    a.max_kv_len = (int32_t)std::min<int64_t>(room, INT32_MAX);
  } else {
    a.max_kv_len = int32(o[7], "max_kv_len");
  }
  a.scale = 1.0f / std::sqrt((float)hq.d);
  if (o[8] != Py_None) {
    a.scale = (float)PyFloat_AsDouble(o[8]);
    if (PyErr_Occurred()) throw Raised{};
  }
  a.causal = truth(o[9]);
  Device dev;
  dev.first(q);
  dev.also(kc);
  dev.also(vc);
  dev.also(bt);
  dev.also(kl);
  dev.also(cu);
  dev.also(given);
  at::Tensor out = given ? *given : empty(q.sizes(), q.scalar_type(), dev.index);
  const Heads ho(out, "out", true);
  a.q = q.data_ptr();
  a.out = out.data_ptr();
  a.q_token_stride = hq.ts; a.q_head_stride = hq.hs; a.out_token_stride = ho.ts; a.out_head_stride = ho.hs;
  a.block_table = bt.data_ptr<int32_t>();
  a.block_table_stride = batch > 1 ? bt.stride(0) : 0;
  a.kv_len = kl.data_ptr<int32_t>();
  a.cu_q = cu.data_ptr<int32_t>();
  a.tokens = hq.n;
  a.heads = (int32_t)hq.h;
  int32_t* words = error_words(dev.index);
  c10::cuda::CUDAGuard guard((c10::DeviceIndex)dev.index);
  const int64_t need = rg_attention_paged_workspace_size(&c, &a);
  at::Tensor space;
  if (need > 0) space = empty({need}, at::kByte, dev.index);
  call(dev.index, [&](void* st) {
    return rg_attention_paged(&c, &a, need > 0 ? space.data_ptr() : nullptr, words, st);
  });
  return THPVariable_Wrap(out);
}

// device -> its error words, or None before its first call
PyObject* words(PyObject* const* o) {
  const long long d = integer(o[0]);
  if (d < 0 || d >= kDevices || !g_words[d].defined()) Py_RETURN_NONE;
  return THPVariable_Wrap(g_words[d]);
}

PyObject* set_check(PyObject* const* o) {
  Py_XINCREF(o[0]);
  Py_XSETREF(g_check, o[0]);
  Py_RETURN_NONE;
}

// A method of N positional arguments whose C++ exceptions become Python's.
template <PyObject* (*F)(PyObject* const*), Py_ssize_t N>
PyObject* method(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != N) {
    PyErr_Format(PyExc_TypeError, "%zd arguments are needed, got %zd", N, n);
    return nullptr;
  }
  try {
    return F(args);
  } catch (const Raised&) {
    return nullptr;
  } catch (const std::invalid_argument& e) {
    PyErr_SetString(PyExc_ValueError, e.what());
  } catch (const c10::OutOfMemoryError& e) {
    PyErr_SetString(PyExc_MemoryError, e.what_without_backtrace());
  } catch (const c10::Error& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

#define RG_METHOD(name, f, n) {name, (PyCFunction)(void (*)(void))method<f, n>, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {RG_METHOD("quantize", quantize, 1),   RG_METHOD("linear", linear, 8),
                         RG_METHOD("rope", rope, 5),           RG_METHOD("append", append, 10),
                         RG_METHOD("attention", attention, 11), RG_METHOD("words", words, 1),
                         RG_METHOD("set_check", set_check, 1), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_serving_bind", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject* PyInit__serving_bind() {
  PyObject* m = PyModule_Create(&module);
  if (m && PyModule_AddStringConstant(m, "torch_version", RG_TORCH_VERSION) < 0) Py_CLEAR(m);
  return m;
}
