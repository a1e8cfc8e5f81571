// paged_q8.cuh -- the paged 8-bit KV cache: page planning, quantising append,
// read-back and causal attention.
#pragma once

#include <cuda_runtime.h>

#include <string>

#include "../../include/fnmoe.h"

namespace fnmoe {

int page_plan(const FnPagePlanArgs *a, cudaStream_t s, std::string &err);
int kv_append_q8(const FnQ8AppendArgs *a, cudaStream_t s, std::string &err);
int kv_read_q8(const FnQ8ReadArgs *a, cudaStream_t s, std::string &err);

int check_q8_cache(const FnQ8Cache &c, std::string &err);
int paged_attention_q8_workspace_size(const FnQ8AttentionArgs *a, uint64_t *bytes, std::string &err);
int paged_attention_q8(const FnQ8AttentionArgs *a, cudaStream_t s, std::string &err);

}  // namespace fnmoe
