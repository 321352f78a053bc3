// Launches of linear_kernels.hip, as linear_bindings.cpp calls them.
#pragma once

#include <hip/hip_runtime_api.h>

#include <cstdint>

// element types
#define ATOMO_F32 0
#define ATOMO_BF16 1
#define ATOMO_F16 2

// activations
#define ATOMO_ACT_NONE 0
#define ATOMO_ACT_RELU 1
#define ATOMO_ACT_GELU 2
#define ATOMO_ACT_SILU 3

// which index of an operand is contiguous in memory
#define ATOMO_FORWARD 0  // both by the reduction:       x, weight
#define ATOMO_GRAD_X 1   // the first by its own index:  weight, dp
#define ATOMO_GRAD_W 2   // both by their own index:     x, dp

// out[j][i] = act(sum_k p(i, k) q(j, k) + bias[i]) + residual[j][i]
struct AtomoProduct {
  const void* p;
  const void* q;
  void* out;
  const void* bias;      // or null
  const void* residual;  // or null
  void* slope;           // act'(.), or null
  int64_t ldp, ldq, ldo, ldr;
  int ni, nj, nk;
  int type, form, act;
};

extern "C" {
void atomo_product_launch(const AtomoProduct* a, hipStream_t stream);
// dp = dy * slope where dp is wanted (slope by relu's output where
// `by_output`), and the sums of dp's columns where db is
void atomo_linear_dp_launch(const void* dy, int64_t ld_dy, const void* slope,
                            int by_output, void* dp, void* db, float* partial,
                            int row_blocks, int rows, int columns, int type,
                            hipStream_t stream);
}
