// The element types of the sequence operators.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "sequence_kernels.h"

namespace mia {

// Calls f with a null pointer to elements of `type`.
template <typename F>
void by_type(SequenceType type, F&& f) {
  if (type == kSeqBf16) f((__nv_bfloat16*)nullptr);
  else if (type == kSeqF16) f((__half*)nullptr);
  else f((float*)nullptr);
}

}  // namespace mia
