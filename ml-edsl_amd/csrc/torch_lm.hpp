// The language-model launches on torch tensors (lm_torch.cpp), METH_FASTCALL.
#pragma once

#define PY_SSIZE_T_CLEAN
#include <Python.h>

PyObject* edsl_torch_rms_norm(PyObject*, PyObject* const* args, Py_ssize_t n);
PyObject* edsl_torch_rms_norm_backward(PyObject*, PyObject* const* args, Py_ssize_t n);
PyObject* edsl_torch_q4_dense(PyObject*, PyObject* const* args, Py_ssize_t n);
PyObject* edsl_torch_token_logprobs(PyObject*, PyObject* const* args, Py_ssize_t n);
PyObject* edsl_torch_token_logprobs_backward(PyObject*, PyObject* const* args, Py_ssize_t n);
