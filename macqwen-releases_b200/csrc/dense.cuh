// dense.cuh -- the dense steps around the block: norms and 8-bit rows, the
// matrix product with its epilogue, and the draw of a token from logits.
#pragma once

#include <cuda_runtime.h>

#include <string>

#include "../../include/fnmoe.h"

namespace fnmoe {

int add_rms_norm(const FnNormArgs *a, cudaStream_t s, std::string &err);
int dequantize_rows(const FnRowCodesArgs *a, cudaStream_t s, std::string &err);
int linear(const FnLinearArgs *a, cudaStream_t s, std::string &err);
int sample(const FnSampleArgs *a, cudaStream_t s, std::string &err);

}  // namespace fnmoe
