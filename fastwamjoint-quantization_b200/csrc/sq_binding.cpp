// CPython front of the block operators for the ordinary call: tensors that are what the kernels read as they are (device,
// dtype, shape, contiguity, alignment), outputs allocated here, no gradient, the current device.  It checks that and
// launches; for anything else it returns None and the Python wrapper of the same name (native.py) takes over, with its
// conversions and its errors.  The smallest calls take 2 to 5 us on the device and took 12 to 17 us of Python.
// The C ABI of libsq_b200.so is what it calls, like the wrappers.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/empty_strided.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <array>
#include <cstring>

#include "../../include/sq_b200.h"

namespace {

using at::Tensor;

struct No {};  // not an ordinary call

const Tensor& tensor_of(PyObject* o) {
  if (!THPVariable_CheckExact(o)) throw No{};
  return THPVariable_Unpack(o);
}

// the call's device: that of its first tensor, which has to be the current one
struct Device {
  c10::Device device;
  bool grad = c10::GradMode::is_enabled();
  explicit Device(const Tensor& t) : device(t.device()) {
    if (!t.is_cuda() || device.index() != c10::cuda::current_device()) throw No{};
  }
  // `t` on this device and without a gradient or a tangent to lose; its address is `align` bytes aligned
  void* take(const Tensor& t, uintptr_t align) const {
    if (t.device() != device || (grad && t.requires_grad()) || t._fw_grad(0).defined() || t.is_conj() || t.is_neg()) throw No{};
    void* p = t.data_ptr();
    if (reinterpret_cast<uintptr_t>(p) & (align - 1)) throw No{};
    return p;
  }
  void* stream() const { return c10::cuda::getCurrentCUDAStream(device.index()).stream(); }
};

int io_dtype(const Tensor& t) {
  if (t.scalar_type() == at::kBFloat16) return SQ_BF16;
  if (t.scalar_type() == at::kHalf) return SQ_FP16;
  throw No{};
}

int choice(PyObject* o, std::initializer_list<std::pair<const char*, int>> names, int none) {
  if (o == Py_None) return none;
  if (!PyUnicode_Check(o)) throw No{};
  for (const auto& [name, value] : names)
    if (PyUnicode_CompareWithASCIIString(o, name) == 0) return value;
  throw No{};
}
int activation_of(PyObject* o) { return choice(o, {{"gelu", SQ_ACT_FN_GELU}}, SQ_ACT_FN_NONE); }
int norm_of(PyObject* o) { return choice(o, {{"rms", SQ_NORM_RMS}, {"layer", SQ_NORM_LAYER}}, SQ_NORM_NONE); }

double number(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    throw No{};
  }
  return v;
}

void need(bool ok) {
  if (!ok) throw No{};
}

// Allocation may wait for the device and a launch for room in its queue: other Python threads run meanwhile.
class NoLock {
 public:
  NoLock() : state_(PyEval_SaveThread()) {}
  ~NoLock() { PyEval_RestoreThread(state_); }
  NoLock(const NoLock&) = delete;
  NoLock& operator=(const NoLock&) = delete;

 private:
  PyThreadState* state_;
};

PyObject* wrap(Tensor t) { return THPVariable_Wrap(std::move(t)); }

struct Weight {
  int64_t n, k;
  const void* codes;
  const float* scales;
  const void* bias;
};
Weight weight_of(const Device& d, PyObject* weight, PyObject* scales, PyObject* bias, at::ScalarType out) {
  const Tensor &w = tensor_of(weight), &s = tensor_of(scales);
  need(w.scalar_type() == at::kFloat8_e4m3fn && w.dim() == 2 && w.is_contiguous());
  Weight r = {w.size(0), w.size(1), d.take(w, 16), nullptr, nullptr};
  need(r.n > 0 && r.n % 8 == 0 && r.k > 0 && r.k % 16 == 0);
  need(s.scalar_type() == at::kFloat && s.dim() == 2 && s.size(0) == (r.n + 127) / 128 && s.size(1) == (r.k + 127) / 128 && s.is_contiguous());
  r.scales = static_cast<const float*>(d.take(s, 4));
  if (bias != Py_None) {
    const Tensor& b = tensor_of(bias);
    need(b.scalar_type() == out && b.dim() == 1 && b.size(0) == r.n && b.is_contiguous());
    r.bias = d.take(b, 2);
  }
  return r;
}

Tensor output_like(const Tensor& x, int64_t n, at::ScalarType dtype) {
  c10::SmallVector<int64_t, 6> shape(x.sizes().begin(), x.sizes().end());
  shape.back() = n;
  return at::empty(shape, x.options().dtype(dtype));
}

// (codes, scales, weight, weight_scales, bias, out_dtype)
PyObject* gemm(PyObject* const* a) {
  const Tensor &x = tensor_of(a[0]), &s = tensor_of(a[1]);
  need(THPDtype_Check(a[5]));
  const at::ScalarType out_type = reinterpret_cast<THPDtype*>(a[5])->scalar_type;
  need((out_type == at::kBFloat16 || out_type == at::kHalf) && x.scalar_type() == at::kFloat8_e4m3fn && x.dim() >= 2 && x.is_contiguous());
  const Device d(x);
  const void* codes = d.take(x, 16);
  const Weight w = weight_of(d, a[2], a[3], a[4], out_type);
  need(x.size(-1) == w.k && x.numel() > 0);
  const int64_t rows = x.numel() / w.k;
  need(s.scalar_type() == at::kFloat && s.dim() == 2 && s.size(0) == rows && s.size(1) == (w.k + 127) / 128);
  const float* scales = static_cast<const float*>(d.take(s, 4));
  Tensor out;
  {
    const NoLock released;
    out = output_like(x, w.n, out_type);
    need(sq_fp8_gemm(codes, scales, s.stride(0), s.stride(1), w.codes, w.scales, w.bias, out.data_ptr(),
                     out_type == at::kBFloat16 ? SQ_BF16 : SQ_FP16, rows, w.n, w.k, d.stream()) == SQ_OK);
  }
  return wrap(std::move(out));
}

// (x, weight, weight_scales, bias, input_activation)
PyObject* linear(PyObject* const* a) {
  const Tensor& x = tensor_of(a[0]);
  const int dtype = io_dtype(x), activation = activation_of(a[4]);
  need(x.dim() >= 2 && x.is_contiguous());
  const Device d(x);
  const void* from = d.take(x, 16);
  const Weight w = weight_of(d, a[1], a[2], a[3], x.scalar_type());
  need(x.size(-1) == w.k && x.numel() > 0);
  const int64_t rows = x.numel() / w.k;
  const size_t bytes = sq_fp8_workspace_bytes(rows, w.k);
  Tensor out;
  {
    const NoLock released;
    const Tensor workspace = at::empty({static_cast<int64_t>(bytes)}, x.options().dtype(at::kByte));
    out = output_like(x, w.n, x.scalar_type());
    need(sq_fp8_linear(from, dtype, rows, w.k, w.n, activation, w.codes, w.scales, w.bias, out.data_ptr(), workspace.data_ptr(),
                       bytes, d.stream()) == SQ_OK);
  }
  return wrap(std::move(out));
}

// rows of parameters (SqParam) that the kernel can read in place
SqParam rows_param(const Device& d, PyObject* o, const Tensor& x, int64_t rows) {
  SqParam q = {};
  if (o == Py_None) return q;
  const Tensor& t = tensor_of(o);
  const bool f32 = t.scalar_type() == at::kFloat;
  const int64_t width = x.size(-1);
  need((f32 || t.scalar_type() == x.scalar_type()) && t.dim() >= 1 && t.size(-1) == width && t.stride(-1) == 1);
  int64_t groups = 1, stride = width;
  if (t.dim() == 2) {
    groups = t.size(0);
    stride = t.stride(0);
  } else if (t.dim() > 2) {
    need(t.is_contiguous());
    groups = t.numel() / width;
  }
  need(groups > 0 && rows % groups == 0 && stride >= 0 && stride % 8 == 0);
  q.data = d.take(t, f32 ? 32 : 16);
  q.row_stride = stride;
  q.span = rows / groups;
  q.is_fp32 = f32;
  return q;
}
SqParam channel_param(const Device& d, PyObject* o, const Tensor& x) {
  SqParam q = {};
  if (o == Py_None) return q;
  const Tensor& t = tensor_of(o);
  const bool f32 = t.scalar_type() == at::kFloat;
  need((f32 || t.scalar_type() == x.scalar_type()) && t.dim() == 1 && t.size(0) == x.size(-1) && t.is_contiguous());
  q.data = d.take(t, f32 ? 32 : 16);
  q.is_fp32 = f32;
  return q;
}

// (x, branch, gate, residual_scale, post_norm, post_weight, post_bias, norm, weight, bias, mod_scale, mod_shift, eps, quantize)
PyObject* block_norm(PyObject* const* a) {
  const Tensor& x = tensor_of(a[0]);
  SqBlockNorm b = {};
  b.dtype = io_dtype(x);
  need(x.dim() >= 2 && x.is_contiguous() && x.numel() > 0 && PyBool_Check(a[13]));
  const bool quantize = a[13] == Py_True, branch = a[1] != Py_None;
  const Device d(x);
  b.x = d.take(x, 16);
  b.width = x.size(-1);
  b.rows = x.numel() / b.width;
  b.post_kind = norm_of(a[4]);
  b.norm_kind = norm_of(a[7]);
  b.residual_scale = static_cast<float>(number(a[3]));
  b.eps = static_cast<float>(number(a[12]));
  need(branch || (b.norm_kind != SQ_NORM_NONE && a[2] == Py_None && b.post_kind == SQ_NORM_NONE && b.residual_scale == 1.0f));
  need(b.norm_kind != SQ_NORM_NONE || (!quantize && a[8] == Py_None && a[9] == Py_None && a[10] == Py_None && a[11] == Py_None));
  need(b.post_kind != SQ_NORM_NONE || (a[5] == Py_None && a[6] == Py_None));
  need(b.width % (quantize ? 16 : 8) == 0 && b.width <= 16384);
  b.gate = rows_param(d, a[2], x, b.rows);
  b.post_weight = channel_param(d, a[5], x);
  b.post_bias = channel_param(d, a[6], x);
  b.weight = channel_param(d, a[8], x);
  b.bias = channel_param(d, a[9], x);
  b.mod_scale = rows_param(d, a[10], x, b.rows);
  b.mod_shift = rows_param(d, a[11], x, b.rows);
  if (branch) {
    const Tensor& t = tensor_of(a[1]);
    need(t.scalar_type() == x.scalar_type() && t.sizes() == x.sizes() && t.is_contiguous());
    b.branch = d.take(t, 16);
  }
  Tensor h, z, scales;
  {
    const NoLock released;
    if (branch) {
      h = at::empty(x.sizes(), x.options());
      b.h_out = h.data_ptr();
    }
    if (b.norm_kind != SQ_NORM_NONE) {
      z = at::empty(x.sizes(), x.options().dtype(quantize ? at::kFloat8_e4m3fn : x.scalar_type()));
      b.z_out = z.data_ptr();
      if (quantize) {
        scales = at::empty_strided({b.rows, (b.width + 127) / 128}, {1, b.rows}, x.options().dtype(at::kFloat));
        b.scales = scales.data_ptr<float>();
        b.scales_row_stride = 1;
        b.scales_group_stride = b.rows;
      }
    }
    need(sq_block_norm(&b, d.stream()) == SQ_OK);
  }
  PyObject* first = a[0];
  if (branch) first = wrap(std::move(h));
  else Py_INCREF(first);
  PyObject* second = Py_None;
  if (b.norm_kind == SQ_NORM_NONE) Py_INCREF(second);
  else if (quantize) second = Py_BuildValue("(NN)", wrap(std::move(z)), wrap(std::move(scales)));
  else second = wrap(std::move(z));
  return Py_BuildValue("(NN)", first, second);
}

struct Heads {
  void* data;
  int64_t strides[3];
};
Heads heads_of(const Device& d, const Tensor& t) {
  need(t.stride(3) == 1 && ((t.stride(0) | t.stride(1) | t.stride(2)) & 7) == 0);
  return {d.take(t, 16), {t.stride(0), t.stride(1), t.stride(2)}};
}
const void* rotary_weight(const Device& d, PyObject* o, const Tensor& q, int64_t count, int norm, int32_t* f32) {
  if (o == Py_None) return nullptr;
  const Tensor& t = tensor_of(o);
  *f32 = t.scalar_type() == at::kFloat;
  need(norm != SQ_ROTARY_NORM_NONE && (*f32 || t.scalar_type() == q.scalar_type()) && t.dim() == 1 && t.is_contiguous() &&
       t.size(0) == (norm == SQ_ROTARY_NORM_TOKEN ? count * q.size(3) : q.size(3)));
  return d.take(t, *f32 ? 32 : 16);
}

// (q, k, positions, inv_freq, sections, layout, norm, q_weight, k_weight, eps)
PyObject* rotary(PyObject* const* a) {
  const Tensor &q = tensor_of(a[0]), &positions = tensor_of(a[2]), &inv_freq = tensor_of(a[3]);
  SqRotary r = {};
  r.dtype = io_dtype(q);
  need(q.dim() == 4 && q.numel() > 0);
  const Device d(q);
  const Heads qh = heads_of(d, q);
  r.q = qh.data;
  std::memcpy(r.q_strides, qh.strides, sizeof(qh.strides));
  r.batch = q.size(0);
  r.length = q.size(1);
  r.heads = static_cast<int32_t>(q.size(2));
  r.dim = static_cast<int32_t>(q.size(3));
  need(q.size(2) <= 4096 && q.size(3) <= 256 && q.size(3) % 8 == 0);
  need(a[5] != Py_None);
  r.layout = choice(a[5], {{"interleaved", SQ_ROTARY_INTERLEAVED}, {"half", SQ_ROTARY_HALF}}, 0);
  r.norm = choice(a[6], {{"head", SQ_ROTARY_NORM_HEAD}, {"token", SQ_ROTARY_NORM_TOKEN}}, SQ_ROTARY_NORM_NONE);
  need(PyTuple_CheckExact(a[4]) && PyTuple_GET_SIZE(a[4]) >= 1 && PyTuple_GET_SIZE(a[4]) <= SQ_ROTARY_AXES);
  r.axes = static_cast<int32_t>(PyTuple_GET_SIZE(a[4]));
  int64_t pairs = 0;
  for (int i = 0; i < r.axes; ++i) {
    const double s = number(PyTuple_GET_ITEM(a[4], i));
    need(s >= 0 && s <= 128 && s == static_cast<int>(s));
    r.sections[i] = static_cast<int32_t>(s);
    pairs += r.sections[i];
  }
  need(pairs >= 1 && 2 * pairs <= r.dim);
  need(inv_freq.scalar_type() == at::kDouble && inv_freq.dim() == 1 && inv_freq.size(0) == pairs && inv_freq.is_contiguous());
  r.inv_freq = static_cast<const double*>(d.take(inv_freq, 8));
  const int64_t pd = positions.dim();
  need((pd == 2 || pd == 3) && positions.size(-1) == r.axes && positions.size(-2) == r.length && positions.stride(-1) == 1 &&
       (pd == 2 || positions.size(0) == 1 || positions.size(0) == r.batch));
  if (positions.scalar_type() == at::kInt) r.position_type = SQ_POS_INT32;
  else if (positions.scalar_type() == at::kLong) r.position_type = SQ_POS_INT64;
  else if (positions.scalar_type() == at::kFloat) r.position_type = SQ_POS_FP32;
  else throw No{};
  r.positions = d.take(positions, r.position_type == SQ_POS_INT64 ? 8 : 4);
  r.position_token_stride = positions.stride(-2);
  r.position_batch_stride = pd == 3 && positions.size(0) > 1 ? positions.stride(0) : 0;
  r.eps = static_cast<float>(number(a[9]));
  r.q_weight = rotary_weight(d, a[7], q, r.heads, r.norm, &r.q_weight_fp32);
  auto dense = [&](int64_t heads, int64_t (&s)[3]) {
    s[2] = r.dim;
    s[1] = heads * r.dim;
    s[0] = r.length * s[1];
  };
  dense(r.heads, r.q_out_strides);
  if (a[1] != Py_None) {
    const Tensor& k = tensor_of(a[1]);
    need(k.dim() == 4 && k.scalar_type() == q.scalar_type() && k.size(0) == r.batch && k.size(1) == r.length && k.size(3) == r.dim &&
         k.size(2) >= 1 && k.size(2) <= 4096);
    const Heads kh = heads_of(d, k);
    r.k = kh.data;
    std::memcpy(r.k_strides, kh.strides, sizeof(kh.strides));
    r.kv_heads = static_cast<int32_t>(k.size(2));
    r.k_weight = rotary_weight(d, a[8], q, r.kv_heads, r.norm, &r.k_weight_fp32);
    dense(r.kv_heads, r.k_out_strides);
  } else {
    need(a[8] == Py_None);
  }
  int64_t lanes = 1;
  while (8 * lanes < r.dim) lanes *= 2;
  need((r.heads + static_cast<int64_t>(r.kv_heads)) * lanes <= 4096);
  Tensor q_out, k_out;
  {
    const NoLock released;
    q_out = at::empty(q.sizes(), q.options());
    r.q_out = q_out.data_ptr();
    if (a[1] != Py_None) {
      k_out = at::empty({r.batch, r.length, r.kv_heads, r.dim}, q.options());
      r.k_out = k_out.data_ptr();
    }
    need(sq_rotary(&r, d.stream()) == SQ_OK);
  }
  PyObject* second = Py_None;
  if (a[1] != Py_None) second = wrap(std::move(k_out));
  else Py_INCREF(second);
  return Py_BuildValue("(NN)", wrap(std::move(q_out)), second);
}

// A C++ exception (an allocation that fails, a dispatcher error) is not this front's to report: the wrapper meets it too
// and raises it with its own message.
template <PyObject* (*kCall)(PyObject* const*), Py_ssize_t kCount>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t count) {
  try {
    if (count == kCount) return kCall(args);
  } catch (const No&) {
  } catch (const std::exception&) {
  }
  PyErr_Clear();
  Py_RETURN_NONE;
}

template <PyObject* (*kCall)(PyObject* const*), Py_ssize_t kCount>
PyCFunction method() {
  return reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&entry<kCall, kCount>));
}

PyMethodDef methods[] = {{"fp8_gemm", method<gemm, 6>(), METH_FASTCALL, nullptr},
                         {"fp8_linear", method<linear, 5>(), METH_FASTCALL, nullptr},
                         {"block_norm", method<block_norm, 14>(), METH_FASTCALL, nullptr},
                         {"rotary", method<rotary, 10>(), METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef definition = {PyModuleDef_HEAD_INIT, "sq_binding", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_sq_binding() { return PyModule_Create(&definition); }
