// Python's way to the operators over lists of tensors.  The dispatcher boxes every tensor of a list
// (156 ns each, 245 us for the four lists of a step over 392 adapters, more than the step takes on
// the GPU); this module unpacks the lists directly.  The functions behind it are the ones that
// torch.ops.mxs_nf4 has (step_lists.h).
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <vector>

#include "step_lists.h"

namespace {

// What the dispatcher would have resolved before a kernel: subclasses that handle operators
// themselves (sharded and fake tensors), negated views, zeros without memory.  Their memory is not
// their values, and there is no dispatcher here to see to it.
bool plain(const at::Tensor& t) {
  constexpr c10::DispatchKeySet odd({c10::DispatchKey::Python, c10::DispatchKey::Negative,
                                     c10::DispatchKey::ZeroTensor,
                                     c10::DispatchKey::Functionalize});
  return !t.key_set().has_any(odd);
}

void check_plain(const at::Tensor& t, const char* name) {
  TORCH_CHECK_VALUE(plain(t), name, " must be a tensor that holds its values itself, got one with ",
                    t.key_set());
}

// The tensors of a Python list, borrowed: the list keeps them alive for the call, so their
// reference counts stay as they are (two atomic operations a tensor saved).
class List {
 public:
  List(PyObject* obj, const char* name) {
    TORCH_CHECK_TYPE(PyList_Check(obj), name, " must be a list of tensors");
    const Py_ssize_t n = PyList_GET_SIZE(obj);
    tensors_.reserve(n);
    for (Py_ssize_t i = 0; i < n; i++) {
      PyObject* x = PyList_GET_ITEM(obj, i);
      bool good = THPVariable_Check(x);
      if (good) {
        const at::Tensor& t = THPVariable_Unpack(x);
        good = t.is_cuda() && plain(t);
        if (good) tensors_.push_back(c10::MaybeOwnedTraits<at::Tensor>::createBorrow(t));
      }
      if (!good) {
        release();
        TORCH_CHECK_TYPE(THPVariable_Check(x), name, "[", i, "] must be a tensor, got ",
                         Py_TYPE(x)->tp_name);
        TORCH_CHECK_VALUE(THPVariable_Unpack(x).is_cuda(), name, "[", i,
                          "] must be a GPU tensor, found ", THPVariable_Unpack(x).device());
        check_plain(THPVariable_Unpack(x), name);
      }
    }
  }
  ~List() { release(); }
  List(const List&) = delete;
  List& operator=(const List&) = delete;
  operator at::TensorList() const { return tensors_; }

 private:
  void release() {
    for (at::Tensor& t : tensors_) c10::MaybeOwnedTraits<at::Tensor>::destroyBorrow(t);
    tensors_.clear();
  }
  std::vector<at::Tensor> tensors_;
};

std::optional<at::Tensor> maybe(PyObject* obj, const char* name) {
  if (obj == Py_None) return std::nullopt;
  TORCH_CHECK_TYPE(THPVariable_Check(obj), name, " must be a tensor or None");
  check_plain(THPVariable_Unpack(obj), name);
  return THPVariable_Unpack(obj);
}

PyObject* grad_norm(PyObject*, PyObject* args) {
  HANDLE_TH_ERRORS
  PyObject *grads, *scale;
  if (!PyArg_ParseTuple(args, "OO", &grads, &scale)) return nullptr;
  const List g(grads, "grads");
  return THPVariable_Wrap(mxs_lists::grad_norm(g, maybe(scale, "grad_scale")));
  END_HANDLE_TH_ERRORS
}

PyObject* adamw_step(PyObject*, PyObject* args) {
  HANDLE_TH_ERRORS
  PyObject *p, *g, *m, *v, *ms, *vs, *step, *lr_dev, *norm, *scale, *found;
  mxs_lists::StepOptions o;
  if (!PyArg_ParseTuple(args, "OOOOOOOdOddddOdOO", &p, &g, &m, &v, &ms, &vs, &step, &o.lr,
                        &lr_dev, &o.beta1, &o.beta2, &o.eps, &o.weight_decay, &norm, &o.max_norm,
                        &scale, &found))
    return nullptr;
  TORCH_CHECK_TYPE(THPVariable_Check(step), "step must be a tensor");
  check_plain(THPVariable_Unpack(step), "step");
  o.lr_dev = maybe(lr_dev, "lr");
  o.norm = maybe(norm, "norm");
  o.grad_scale = maybe(scale, "grad_scale");
  o.found_inf = maybe(found, "found_inf");
  const List params(p, "params"), grads(g, "grads"), avgs(m, "exp_avgs"),
      avg_sqs(v, "exp_avg_sqs"), scales(ms, "exp_avg_scales"), sq_scales(vs, "exp_avg_sq_scales");
  mxs_lists::adamw_step(params, grads, avgs, avg_sqs, scales, sq_scales, THPVariable_Unpack(step),
                        o);
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {{"grad_norm", grad_norm, METH_VARARGS, nullptr},
                         {"adamw_step", adamw_step, METH_VARARGS, nullptr},
                         {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_mxs_lists", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__mxs_lists() { return PyModule_Create(&module); }
