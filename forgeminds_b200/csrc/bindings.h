// What the files of Python bindings share.
#pragma once
#include <pybind11/pybind11.h>

void fmb_count_launches(int kernels);               // bindings.cpp keeps the count of enqueued kernels
void fmb_bind_rows(pybind11::module_& m);           // bindings_rows.cpp
