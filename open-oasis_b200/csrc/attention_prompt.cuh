// Arguments of the packed causal attention kernels.
#pragma once
#include <cuda_runtime.h>

namespace oasis {

struct PromptParams {
  const void *q, *k, *v;
  void* out;
  long long q_row, q_head, k_row, k_head, v_row, v_head, o_row, o_head;  // elements
  int rows;  // rows of every operand
  const int* cu;
  int n, longest, heads, kv_heads, head_dim, dtype;
  float scale_log2;  // scale / ln 2
};

int prompt_rows_launch(const PromptParams& p, cudaStream_t s);
int prompt_tc_launch(const PromptParams& p, cudaStream_t s);
int read_device_error_prompt(int reset);

}  // namespace oasis
