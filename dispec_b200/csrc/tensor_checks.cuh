// Checks of described tensors (tensor_desc.h) at the C entry points.
#pragma once
#include "common.cuh"
#include "tensor_desc.h"

// contiguous, of this type and device, with these sizes
inline bool tensor_is(const DspTensor& t, int dtype, int device, int dims, long a = 0, long b = 0) {
  return t.dtype == dtype && t.device == device && t.dims == dims && t.contiguous && (dims < 1 || t.size[0] == a) &&
         (dims < 2 || t.size[1] == b);
}
// a page table of at least `seqs` rows, neighbouring pages side by side
inline bool is_page_table(const DspTensor& t, int device, long seqs) {
  return t.dtype == DSP_T_I32 && t.device == device && t.dims == 2 && t.size[0] >= seqs && t.stride[1] == 1;
}
