// The calls of a decode step on torch tensors, append and attention, without Python's cost per tensor
// attribute.  Appending one row, back to back: 14.7 us a call packed in Python, 3.5 here, of which the launch
// takes most; one row's attention 10.9 and 9.2, where the kernel takes 8.6.
//
// Both functions look at their arguments as paged.py does.  What is in order is packed and called;
// for anything else they return None before calling, and paged.py goes through the arguments itself and
// says what is wrong.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/llx.h"

namespace {

constexpr auto kI8 = at::kChar;
constexpr auto kI16 = at::kShort;
constexpr auto kI32 = at::kInt;

struct Unusual {};  // for paged.py to look at

void need(bool ok) {
  if (!ok) throw Unusual();
}

class Args {
 public:
  Args(PyObject* const* args, Py_ssize_t n, Py_ssize_t want) : args_(args) { need(n == want); }

  // the next argument: a tensor of `type` on the call's device (the first tensor's)
  const at::Tensor& tensor(at::ScalarType type) {
    PyObject* o = args_[at_++];
    need(THPVariable_Check(o));
    const at::Tensor& t = THPVariable_Unpack(o);
    need(t.defined() && t.layout() == at::kStrided && t.is_cuda() && t.scalar_type() == type);
    if (device_ < 0) device_ = t.get_device();
    need(t.get_device() == device_);
    return t;
  }
  const at::Tensor* maybe(at::ScalarType type) {
    if (args_[at_] != Py_None) return &tensor(type);
    ++at_;
    return nullptr;
  }
  int64_t number() { return number(args_[at_++]); }
  void pair(int64_t& a, int64_t& b) {
    PyObject* o = args_[at_++];
    need(PyTuple_Check(o) && PyTuple_GET_SIZE(o) == 2);
    a = number(PyTuple_GET_ITEM(o, 0));
    b = number(PyTuple_GET_ITEM(o, 1));
  }
  // (gamma, eps, C, shift) of a norm, or None
  void norm(int64_t dim, const int16_t*& gamma, int64_t& eps, int64_t& C, int64_t& shift) {
    PyObject* o = args_[at_];
    gamma = nullptr;
    eps = C = shift = 0;
    if (o == Py_None) {
      ++at_;
      return;
    }
    need(PyTuple_Check(o) && PyTuple_GET_SIZE(o) == 4);
    Args in(&PyTuple_GET_ITEM(o, 0), 1, 1);
    in.device_ = device_;
    const at::Tensor& g = in.tensor(kI16);
    need(g.dim() == 1 && g.size(0) == dim && (dim <= 1 || g.stride(0) == 1));
    gamma = static_cast<const int16_t*>(g.const_data_ptr());
    eps = number(PyTuple_GET_ITEM(o, 1));
    C = number(PyTuple_GET_ITEM(o, 2));
    shift = number(PyTuple_GET_ITEM(o, 3));
    ++at_;
  }
  int64_t device() const { return device_; }

 private:
  static int64_t number(PyObject* o) {
    need(PyLong_CheckExact(o));
    int over = 0;
    const long long v = PyLong_AsLongLongAndOverflow(o, &over);
    need(!over);
    return v;
  }

  PyObject* const* args_;
  Py_ssize_t at_ = 0;
  int64_t device_ = -1;
};

// row stride of a [rows, heads, dim] tensor whose rows are dense
int64_t row_stride(const at::Tensor& t, int64_t rows, int64_t heads, int64_t dim) {
  need(t.dim() == 3 && t.size(0) == rows && t.size(1) == heads && t.size(2) == dim && t.stride(2) == 1 && t.stride(1) == dim);
  return rows > 1 ? t.stride(0) : heads * dim;
}

template <class A>
void put_pages(A& a, const at::Tensor& k, const at::Tensor& v, int64_t dim) {
  need(k.dim() == 4 && k.sizes() == v.sizes() && k.strides() == v.strides());
  const int64_t P = k.size(2);
  need(k.size(3) == dim && k.stride(3) == 1 && k.stride(2) == dim && k.stride(1) == dim * P);
  a.k_pages = static_cast<decltype(a.k_pages)>(k.data_ptr());
  a.v_pages = static_cast<decltype(a.v_pages)>(v.data_ptr());
  a.page_stride = k.stride(0);
  a.n_pages = k.size(0);
  a.n_kv_heads = k.size(1);
  a.page_size = P;
}

const int32_t* vector(const at::Tensor& t, int64_t n) {
  need(t.dim() == 1 && t.size(0) == n && (n <= 1 || t.stride(0) == 1));
  return static_cast<const int32_t*>(t.const_data_ptr());
}

template <class A>
void put_launch(A& a, const at::Tensor& table, const at::Tensor& length, const at::Tensor& q_start, const at::Tensor* seqs,
                const at::Tensor* status) {
  need(table.dim() == 2 && (table.size(1) <= 1 || table.stride(1) == 1));
  a.table = static_cast<const int32_t*>(table.const_data_ptr());
  a.max_seqs = table.size(0);
  a.max_pages = table.size(1);
  a.table_stride = a.max_seqs > 1 ? table.stride(0) : a.max_pages;
  a.length = vector(length, a.max_seqs);
  need(q_start.dim() == 1 && q_start.size(0) >= 1);
  a.n_seqs = q_start.size(0) - 1;
  a.q_start = vector(q_start, a.n_seqs + 1);
  a.seqs = seqs ? vector(*seqs, a.n_seqs) : nullptr;
  need(seqs || a.n_seqs <= a.max_seqs);
  a.status = status ? static_cast<int32_t*>(status->data_ptr()) : nullptr;
}

// what `fill` packs, called on its device's current stream; None if `fill` finds something unusual
template <class A, class Fill>
PyObject* run(PyObject* const* args, Py_ssize_t n, Py_ssize_t want, Fill fill) {
  try {
    Args in(args, n, want);
    const auto call = reinterpret_cast<llx_status (*)(const A*, void*)>(in.number());
    A a = {};
    fill(in, a);
    a.device = in.device();
    void* stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)a.device).stream();
    llx_status code;
    Py_BEGIN_ALLOW_THREADS;
    code = call(&a, stream);
    Py_END_ALLOW_THREADS;
    return PyLong_FromLong(code);
  } catch (...) {
    PyErr_Clear();
    Py_RETURN_NONE;
  }
}

PyObject* append(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return run<llx_paged_append_args>(args, n, 18, [](Args& in, llx_paged_append_args& a) {
    const at::Tensor &q = in.tensor(kI16), &k = in.tensor(kI16), &v = in.tensor(kI8), &kp = in.tensor(kI8), &vp = in.tensor(kI8);
    const at::Tensor &table = in.tensor(kI32), &length = in.tensor(kI32), &q_start = in.tensor(kI32);
    const at::Tensor &cos = in.tensor(kI16), &sin = in.tensor(kI16);
    need(q.dim() == 3 && q.size(0) > 0);  // tensors without rows have no addresses
    const int64_t R = q.size(0), H = q.size(1), D = q.size(2);
    in.pair(a.q_M, a.q_S);
    in.pair(a.k_M, a.k_S);
    in.norm(D, a.q_gamma, a.q_eps, a.q_C, a.q_shift);
    in.norm(D, a.k_gamma, a.k_eps, a.k_C, a.k_shift);
    const at::Tensor* seqs = in.maybe(kI32);
    const at::Tensor& out = in.tensor(kI8);
    const at::Tensor* status = in.maybe(kI32);
    put_pages(a, kp, vp, D);
    put_launch(a, table, length, q_start, seqs, status);
    need(cos.dim() == 2 && cos.sizes() == sin.sizes() && cos.size(1) == D / 2 && cos.is_contiguous() && sin.is_contiguous());
    a.q = static_cast<const int16_t*>(q.const_data_ptr());
    a.k = static_cast<const int16_t*>(k.const_data_ptr());
    a.v = static_cast<const int8_t*>(v.const_data_ptr());
    a.q8 = static_cast<int8_t*>(out.data_ptr());
    a.cos = static_cast<const int16_t*>(cos.const_data_ptr());
    a.sin = static_cast<const int16_t*>(sin.const_data_ptr());
    a.n_positions = cos.size(0);
    a.rows = R;
    a.n_heads = H;
    a.head_dim = D;
    a.q_stride = row_stride(q, R, H, D);
    a.k_stride = row_stride(k, R, a.n_kv_heads, D);
    a.v_stride = row_stride(v, R, a.n_kv_heads, D);
    a.q8_stride = row_stride(out, R, H, D);
  });
}

PyObject* attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return run<llx_paged_attention_args>(args, n, 15, [](Args& in, llx_paged_attention_args& a) {
    const at::Tensor &q8 = in.tensor(kI8), &kp = in.tensor(kI8), &vp = in.tensor(kI8);
    const at::Tensor &table = in.tensor(kI32), &length = in.tensor(kI32), &q_start = in.tensor(kI32);
    in.pair(a.Ms, a.Ss);
    in.pair(a.Mo, a.So);
    a.prob_bits = in.number();
    a.max_rows = in.number();
    a.max_len = in.number();
    const at::Tensor* seqs = in.maybe(kI32);
    const at::Tensor& out = in.tensor(kI8);
    const at::Tensor* status = in.maybe(kI32);
    need(q8.dim() == 3 && q8.size(0) > 0);
    const int64_t R = q8.size(0), H = q8.size(1), D = q8.size(2);
    put_pages(a, kp, vp, D);
    put_launch(a, table, length, q_start, seqs, status);
    a.q8 = static_cast<const int8_t*>(q8.const_data_ptr());
    a.out = static_cast<int8_t*>(out.data_ptr());
    a.rows = R;
    a.n_heads = H;
    a.head_dim = D;
    a.q8_stride = row_stride(q8, R, H, D);
    a.out_stride = row_stride(out, R, H, D);
  });
}

PyMethodDef methods[] = {
    {"append", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(append)), METH_FASTCALL,
     "append(llx_paged_append's address, paged.append's arguments) -> code, or None"},
    {"attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(attention)), METH_FASTCALL,
     "attention(llx_paged_attention's address, paged.attention's arguments) -> code, or None"},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "torch_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_torch_calls() { return PyModule_Create(&module); }
