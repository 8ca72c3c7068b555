// uv_prompt.h -- launcher of the attention over whole prompts (internal).
#pragma once

#include "uv_kv.h"

namespace uvb {
namespace prompt {

struct Args {
  kv::Strided q, k, v;
  const int32_t *starts_q, *starts_k;  // n + 1 each
  int n, rows_q, rows_k, q_heads, heads, D;
  bool causal, bf16;
  float scale;
  void *out;   // rows_q x q_heads x D, dense
  float *lse;  // rows_q x q_heads, or null
};
cudaError_t launch(const Args &a, cudaStream_t st);

}  // namespace prompt
}  // namespace uvb
