// The operators' functions of the binding (ps_ops_binding.cpp).
#ifndef PS_OPS_BINDING_H
#define PS_OPS_BINDING_H

PyObject* ps_ops_use(PyObject*, PyObject* const* args, Py_ssize_t n);
PyObject* ps_ops_heads(PyObject*, PyObject* const* args, Py_ssize_t n);
PyObject* ps_ops_top(PyObject*, PyObject* const* args, Py_ssize_t n);
PyObject* ps_ops_distill(PyObject*, PyObject* const* args, Py_ssize_t n);

#endif  // PS_OPS_BINDING_H
