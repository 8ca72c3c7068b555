// uv_kv.h -- launchers of the cache held in 4 bits and of the prompt
// attention (internal).
#pragma once

#include "uv_kv.cuh"

namespace uvb {
namespace kv {

// A packed operand of rows x heads x D: element strides of a row and a head.
struct Strided {
  const void *p;
  int64_t row, head;
};

cudaError_t extend_launch(const Cache &c, const int32_t *seqs, const int32_t *counts, int n,
                          int sms, cudaStream_t st);
cudaError_t copy_launch(const Cache &c, const int32_t *src, const int32_t *dst, int n, int sms,
                        cudaStream_t st);
cudaError_t fork_launch(const Cache &c, const int32_t *src, const int32_t *dst,
                        const int32_t *lens, int n, cudaStream_t st);
cudaError_t truncate_launch(const Cache &c, const int32_t *seqs, const int32_t *lens, int n,
                            cudaStream_t st);
cudaError_t compact_launch(const Cache &c, int sms, cudaStream_t st);
cudaError_t recount_launch(const Cache &c, cudaStream_t st);

cudaError_t append_launch(const Cache &c, int layer, const Rows &rows, const Strided &k,
                          const Strided &v, bool bf16, cudaStream_t st);
cudaError_t read_launch(const Cache &c, int layer, const Rows &rows, void *k, void *v, bool bf16,
                        cudaStream_t st);

// The attention's launch shape: columns of one tile and the scratch it takes.
struct AttendPlan {
  int cols = 0;          // (token, head of the group) pairs a block holds
  int64_t jobs = 0;      // upper bound on (sequence, column tile, head)
  int sms = 0;
  int64_t bytes = 0;     // scratch
};
AttendPlan attend_plan(const Cache &c, int n, int rows, int most, int q_heads, int sms);
struct AttendArgs {
  Strided q;
  void *out;       // rows x q_heads x D, dense
  float *lse;      // rows x q_heads, or null
  int q_heads;
  float scale;
  void *scratch;
  unsigned long long call;  // a number that no other call has, not 0
};
cudaError_t attend_launch(const Cache &c, int layer, const Rows &rows, const AttendArgs &a,
                          const AttendPlan &plan, bool bf16, cudaStream_t st);

}  // namespace kv
}  // namespace uvb
