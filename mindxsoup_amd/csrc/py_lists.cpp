// Python's way to the operators over lists of tensors.  The dispatcher boxes every tensor of a list
// (156 ns each, 245 us for the four lists of a step over 392 adapters, more than the step takes on
// the GPU); this module unpacks the lists directly.  The functions behind it are the ones that
// torch.ops.mxs_nf4 has (step_lists.h).
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <vector>

#include "step_lists.h"

namespace {

std::vector<at::Tensor> list(PyObject* obj, const char* name) {
  TORCH_CHECK_TYPE(PyList_Check(obj), name, " must be a list of tensors");
  const Py_ssize_t n = PyList_GET_SIZE(obj);
  std::vector<at::Tensor> out;
  out.reserve(n);
  for (Py_ssize_t i = 0; i < n; i++) {
    PyObject* x = PyList_GET_ITEM(obj, i);
    TORCH_CHECK_TYPE(THPVariable_Check(x), name, "[", i, "] must be a tensor, got ",
                     Py_TYPE(x)->tp_name);
    const at::Tensor& t = THPVariable_Unpack(x);
    TORCH_CHECK_VALUE(t.is_cuda(), name, "[", i, "] must be a GPU tensor, found ", t.device());
    out.push_back(t);
  }
  return out;
}

std::optional<at::Tensor> maybe(PyObject* obj, const char* name) {
  if (obj == Py_None) return std::nullopt;
  TORCH_CHECK_TYPE(THPVariable_Check(obj), name, " must be a tensor or None");
  return THPVariable_Unpack(obj);
}

PyObject* grad_norm(PyObject*, PyObject* args) {
  HANDLE_TH_ERRORS
  PyObject *grads, *scale;
  if (!PyArg_ParseTuple(args, "OO", &grads, &scale)) return nullptr;
  return THPVariable_Wrap(mxs_lists::grad_norm(list(grads, "grads"), maybe(scale, "grad_scale")));
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
  o.lr_dev = maybe(lr_dev, "lr");
  o.norm = maybe(norm, "norm");
  o.grad_scale = maybe(scale, "grad_scale");
  o.found_inf = maybe(found, "found_inf");
  mxs_lists::adamw_step(list(p, "params"), list(g, "grads"), list(m, "exp_avgs"),
                        list(v, "exp_avg_sqs"), list(ms, "exp_avg_scales"),
                        list(vs, "exp_avg_sq_scales"), THPVariable_Unpack(step), o);
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {{"grad_norm", grad_norm, METH_VARARGS, nullptr},
                         {"adamw_step", adamw_step, METH_VARARGS, nullptr},
                         {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_mxs_lists", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__mxs_lists() { return PyModule_Create(&module); }
