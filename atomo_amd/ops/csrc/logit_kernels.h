// Launches of logit_kernels.hip, as logit_bindings.cpp calls them.
#pragma once

#include <hip/hip_runtime_api.h>

#include <cstdint>

// the most alternatives, and the most teacher's entries, of one row
#define ATOMO_LOGIT_TOP_MAX 128
// the most parts of one row
#define ATOMO_LOGIT_MAX_SPLITS 64
// up to here a kernel counts the rows of a mean by itself: a wave reads at
// most 8 KB of labels more, which costs less than one more launch (2 us)
#define ATOMO_LOGIT_COUNT_ROWS 1024

// element types of the logits
#define ATOMO_F32 0
#define ATOMO_BF16 1
#define ATOMO_F16 2

struct AtomoLogprobs {
  const void* logits;
  const int64_t* labels;  // or null
  float* logprob;
  float* entropy;
  float* top_logprob;
  int64_t* top_index;
  // of each part, where there are several: m, S, T and the best keys
  float* part_stat;
  int64_t* part_keys;
  int64_t row_stride, rows, ignore;
  int type, classes, top, splits, part_size;
};

struct AtomoDistill {
  const void* logits;
  const float* values;   // (rows, k)
  const int64_t* index;  // (rows, k)
  const int64_t* labels; // or null
  float* row_loss;
  float* stats;          // (rows, splits, 3): m, S, S_t
  const float* inverse;  // one over the counted rows, or null:
  const float* up;       // the loss's gradient, one or one a row
  void* grad;
  int64_t row_stride, rows, ignore;
  float tau, inv_tau;
  float weight, rest;    // of the teacher (0 only where k is) and of the labels
  float factor;          // then this, unless the kernel is to
  int count;             // count them itself
  int type, classes, k;
  int mode;              // one of ATOMO_DISTILL_*
  int splits, part_size; // of the sums
  int grad_splits, grad_part;
  int up_per_row;
  int skip_one;          // leave the gradient alone where `up` is 1
};

// how exp(d) comes from exp(d / tau): not needed, tau 1, 2, 4, any
#define ATOMO_DISTILL_SOFT 0
#define ATOMO_DISTILL_TAU1 1
#define ATOMO_DISTILL_TAU2 2
#define ATOMO_DISTILL_TAU4 3
#define ATOMO_DISTILL_ANY 4

extern "C" {
// into how many parts, of which size, a row is split
int atomo_logit_splits(int64_t rows, int classes, int type, int* part_size);
void atomo_label_logprobs_launch(const AtomoLogprobs* a, hipStream_t stream);

// whether loss and gradient are computed together, in one read of the logits
int atomo_distill_fits(int64_t rows, int classes, int type);
// whether one wave's registers hold a row
int atomo_distill_short(int classes, int type);
void atomo_distill_fused_launch(const AtomoDistill* a, hipStream_t stream);
void atomo_distill_count_launch(const int64_t* labels, int64_t rows,
                                int64_t ignore, float* inverse,
                                hipStream_t stream);
void atomo_distill_loss_launch(const AtomoDistill* a, hipStream_t stream);
void atomo_distill_sum_launch(const AtomoDistill* a, float* loss,
                              hipStream_t stream);
void atomo_distill_grad_launch(const AtomoDistill* a, hipStream_t stream);
}
