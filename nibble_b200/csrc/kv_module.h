// Python entry points of the 8-bit key/value cache and of rotary positions (kv_module.cpp), for the extension module's table.
#pragma once

#include <Python.h>

namespace w4a16 {

PyObject* rotary(PyObject*, PyObject* const* args, Py_ssize_t count);
PyObject* kv8_bytes(PyObject*, PyObject* const* args, Py_ssize_t count);
PyObject* kv8_append(PyObject*, PyObject* const* args, Py_ssize_t count);
PyObject* kv8_read(PyObject*, PyObject* const* args, Py_ssize_t count);
PyObject* kv8_attention(PyObject*, PyObject* const* args, Py_ssize_t count);

}  // namespace w4a16
