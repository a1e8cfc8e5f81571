// dense.cuh -- the dense steps around the block: norms and 8-bit rows, the
// matrix product with its epilogue, and the draw of a token from logits.
#pragma once

#include <cuda_runtime.h>

#include <string>

#include "../../include/fnmoe.h"

namespace fnmoe {

// Bytes of a caller's array, for refusing outputs that overlap inputs.
struct Span {
  const void *at;
  uint64_t bytes;
  bool meets(const Span &o) const {
    const uint64_t a = reinterpret_cast<uintptr_t>(at), b = reinterpret_cast<uintptr_t>(o.at);
    return at != nullptr && o.at != nullptr && a < b + o.bytes && b < a + bytes;
  }
};

int add_rms_norm(const FnNormArgs *a, cudaStream_t s, std::string &err);
int dequantize_rows(const FnRowCodesArgs *a, cudaStream_t s, std::string &err);
int linear(const FnLinearArgs *a, cudaStream_t s, std::string &err);
int sample(const FnSampleArgs *a, cudaStream_t s, std::string &err);

}  // namespace fnmoe
