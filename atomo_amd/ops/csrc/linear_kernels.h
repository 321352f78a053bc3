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

// how a product is computed: tiles of that size, or a wave for a few columns
#define ATOMO_PLAN_64 0
#define ATOMO_PLAN_128 1
#define ATOMO_PLAN_256 2
#define ATOMO_PLAN_FEW_ROWS 3
#define ATOMO_PLAN_TINY 4

// out[j][i] = act(sum_k p(i, k) q(j, k) + bias[i]) + residual[j][i]
struct AtomoProduct {
  const void* p;
  const void* q;
  void* out;
  const void* bias;      // or null
  const void* residual;  // or null
  void* slope;           // act'(.) in fp32, or null
  float* partial;        // (splits, nj, ld_part), where splits > 1
  int64_t ldp, ldq, ldo, ldr, ld_part;
  int ni, nj, nk;
  int type, form, act;
  // by atomo_product_plan, from type, form, act, p, q, ldp, ldq, the sizes and
  // which of bias, residual and slope there are; `bare`: the tiles have no
  // epilogue, `direct`: operands are loaded straight into LDS
  int plan, splits, k_part, bare, direct;
};

// dp = dy * slope, where dp is wanted; db, the sums of its columns, likewise.
// Without a slope dp is dy; with `by_output` the slope is relu's output, in the
// operands' type, otherwise it is fp32.
struct AtomoLinearDp {
  const void* dy;
  const void* slope;
  void* dp;
  void* db;
  float* partial;  // (row_blocks, columns), where row_blocks > 1
  int64_t ld_dy;
  int by_output, rows, columns, row_blocks, block_rows, type;
};

extern "C" {
void atomo_product_plan(AtomoProduct* a);
void atomo_product_launch(const AtomoProduct* a, hipStream_t stream);
void atomo_linear_dp_launch(const AtomoLinearDp* a, hipStream_t stream);
}
