// Bindings of the operators over sequences: sequence_ops.cpp adds them to the module that bindings.cpp defines.
#pragma once
#include <cuda_runtime.h>
#include <torch/extension.h>

void bind_sequence_ops(pybind11::module& m);

// The current stream of the current device, counted as the launch of one kernel.  Defined in bindings.cpp.
cudaStream_t counted_stream();
void count_launches(int n);
