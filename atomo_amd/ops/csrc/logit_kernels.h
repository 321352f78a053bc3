// Launches of logit_kernels.hip, as logit_bindings.cpp calls them.
#pragma once

#include <hip/hip_runtime_api.h>

#include <cstdint>

// the most alternatives, and the most teacher's entries, of one row
#define ATOMO_LOGIT_TOP_MAX 128

// element types of the logits
#define ATOMO_F32 0
#define ATOMO_BF16 1
#define ATOMO_F16 2

extern "C" {
void atomo_label_logprobs_launch(const void* logits, int type,
                                 int64_t row_stride, int64_t rows, int classes,
                                 const int64_t* labels, int64_t ignore,
                                 int top, float* logprob, float* entropy,
                                 float* top_logprob, int64_t* top_index,
                                 hipStream_t stream);
void atomo_distill_count_launch(const int64_t* labels, int64_t rows,
                                int64_t ignore, float* inverse,
                                hipStream_t stream);
void atomo_distill_loss_launch(const void* logits, int type, int64_t row_stride,
                               int64_t rows, int classes, const float* values,
                               const int64_t* index, int k,
                               const int64_t* labels, int64_t ignore, float tau,
                               float weight, float* row_loss, float* stats,
                               hipStream_t stream);
void atomo_distill_sum_launch(const float* row_loss, int64_t rows,
                              const float* inverse, float factor, float* loss,
                              hipStream_t stream);
void atomo_distill_grad_launch(const void* logits, int type, int64_t row_stride,
                               int64_t rows, int classes, const float* values,
                               const int64_t* index, int k,
                               const int64_t* labels, int64_t ignore, float tau,
                               float weight, const float* stats,
                               const float* up, int up_per_row,
                               const float* inverse, float factor, void* grad,
                               hipStream_t stream);
}
