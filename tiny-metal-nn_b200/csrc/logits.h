// logits.h -- row-wise operators over class logits (logits.cu): log
// probabilities of given tokens with entropy and top alternatives, their
// backward pass, and distillation from a teacher's top logits.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/tmnn_cuda.h"

namespace tmnn {

// Largest number of classes of a row, and of alternatives / teacher entries.
constexpr uint32_t kMaxClasses = 1u << 19;
constexpr uint32_t kMaxTop = 128;

struct LogprobOut {
  float *logprob;       // [n], needs tokens
  float *entropy;       // [n]
  int32_t *top_ids;     // [n x top_k]
  float *top_logprobs;  // [n x top_k]
  float *stats;         // [n x 3]
};

// The checks of the calls below alone (std::invalid_argument), for callers that
// queue other work before.
void check_token_logprobs(const tmnn_logits &x, const void *tokens,
                          int index_type, uint32_t top_k, const LogprobOut &o);
void check_distill(const tmnn_logits &x, const void *ids, int index_type,
                   const void *teacher, int teacher_dtype, uint32_t k,
                   const float *row_weight, const float *loss,
                   const void *d_logits, int64_t d_stride);

// Each checks its arguments (std::invalid_argument) and queues its kernel on
// `st`, which belongs to the current device.  Nothing is allocated and the
// host does not wait, so the calls can be captured.  They return the number
// of kernels launched.
int launch_token_logprobs(const tmnn_logits &x, const void *tokens,
                          int index_type, uint32_t top_k, const LogprobOut &o,
                          cudaStream_t st);
int launch_token_logprobs_backward(const tmnn_logits &x, const void *tokens,
                                   int index_type, const float *stats,
                                   const float *d_logprob,
                                   const float *d_entropy, void *d_logits,
                                   int64_t d_stride, cudaStream_t st);
// row_weight null: every row weighs `weight`.  d_logits null: the loss only.
int launch_distill(const tmnn_logits &x, const void *ids, int index_type,
                   const void *teacher, int teacher_dtype, uint32_t k,
                   const float *row_weight, float weight, float *loss,
                   void *d_logits, int64_t d_stride, cudaStream_t st);
// *sum = the sum of n values in 64 bits, in one fixed order.
void launch_row_sum(const float *values, uint32_t n, double *sum,
                    cudaStream_t st);

}  // namespace tmnn
