// The Python functions of torch_batch.cpp, for the module's table.
#pragma once

#include <Python.h>

namespace spectra_torch {

PyObject* py_axes_append(PyObject*, PyObject* const* args, Py_ssize_t n);
PyObject* py_key_bounds(PyObject*, PyObject* const* args, Py_ssize_t n);
PyObject* py_bounds_values(PyObject*, PyObject* const* args, Py_ssize_t n);
PyObject* py_select(PyObject*, PyObject* const* args, Py_ssize_t n);
PyObject* py_attend_blocks(PyObject*, PyObject* const* args, Py_ssize_t n);
PyObject* py_adjust_logits(PyObject*, PyObject* const* args, Py_ssize_t n);
PyObject* py_next_tokens(PyObject*, PyObject* const* args, Py_ssize_t n);

}  // namespace spectra_torch
