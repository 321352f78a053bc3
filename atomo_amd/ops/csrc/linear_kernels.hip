// Matrix product with bias, activation and residual in its epilogue, forward
// and backward, for MI355X (gfx950).
//
//   forward    y  = act(x W^T + b) + r       x (M, K), W (N, K)
//   backward   dp = dy act'(.)               dr = dy
//              dx = dp W                     dW = dp^T x       db = sum dp
//
// All three products are one kernel, out[j][i] = sum_k p(i, k) q(j, k): they
// differ in which index of p and q is contiguous in memory.  Tiles go through
// registers into LDS, always as rows of the reduction: an operand that lies
// the other way is transposed in registers on the way, in 4 x 4 blocks (fp32:
// a renaming) or 8 x 4 blocks (16-bit: one byte permute for two elements).
// So the inner loop is the same for all: a 16-byte read for each fragment,
// which one 16-bit matrix instruction consumes (k = 16) or four fp32 ones
// (k = 2 each; the order of a sum's terms is free, so lane halves take four
// neighbouring k each).  p gives the rows of the matrix instruction's result:
// a lane then holds four neighbouring i of one j, and stores them at once.
//
// Sums are fp32; an output is rounded once.

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include <cstdint>

#include "linear_kernels.h"

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// memory vectors at the alignment of their elements: rows may be odd
typedef u32x4 u32x4_a4 __attribute__((aligned(4)));
typedef u32x4 u32x4_a2 __attribute__((aligned(2)));
typedef u32x2 u32x2_a2 __attribute__((aligned(2)));

struct F32 {
  using Raw = uint32_t;
  static constexpr int kChunk = 4;  // elements in 16 bytes
  __device__ static float widen(Raw r) { return __uint_as_float(r); }
  __device__ static Raw narrow(float f) { return __float_as_uint(f); }
};
struct BF16 {
  using Raw = uint16_t;
  static constexpr int kChunk = 8;
  __device__ static float widen(Raw r) {
    return __uint_as_float((uint32_t)r << 16);
  }
  __device__ static Raw narrow(float f) {
    return __builtin_bit_cast(Raw, (__bf16)f);
  }
};
struct F16 {
  using Raw = uint16_t;
  static constexpr int kChunk = 8;
  __device__ static float widen(Raw r) {
    return (float)__builtin_bit_cast(_Float16, r);
  }
  __device__ static Raw narrow(float f) {
    return __builtin_bit_cast(Raw, (_Float16)f);
  }
};

template <typename E>
__device__ __forceinline__ void multiply(const u32x4& p, const u32x4& q,
                                         f32x16& acc);
template <>
__device__ __forceinline__ void multiply<BF16>(const u32x4& p, const u32x4& q,
                                               f32x16& acc) {
  acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
      __builtin_bit_cast(bf16x8, p), __builtin_bit_cast(bf16x8, q), acc, 0, 0, 0);
}
template <>
__device__ __forceinline__ void multiply<F16>(const u32x4& p, const u32x4& q,
                                              f32x16& acc) {
  acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(
      __builtin_bit_cast(f16x8, p), __builtin_bit_cast(f16x8, q), acc, 0, 0, 0);
}
template <>
__device__ __forceinline__ void multiply<F32>(const u32x4& p, const u32x4& q,
                                              f32x16& acc) {
#pragma unroll
  for (int c = 0; c < 4; ++c)
    acc = __builtin_amdgcn_mfma_f32_32x32x2f32(
        __uint_as_float(p[c]), __uint_as_float(q[c]), acc, 0, 0, 0);
}

// y and dy/dh of the activation at h
__device__ __forceinline__ float activate(int act, float h, float* slope) {
  if (act == ATOMO_ACT_RELU) {
    // not (h <= 0): NaN passes
    *slope = h <= 0.f ? 0.f : 1.f;
    return h <= 0.f ? 0.f : h;
  }
  if (act == ATOMO_ACT_GELU) {
    const float cdf = 0.5f * erfcf(h * -0.70710678118654752f);
    const float pdf = 0.39894228040143268f * expf(-0.5f * h * h);
    *slope = h == -__builtin_huge_valf() ? 0.f : cdf + (pdf > 0.f ? h * pdf : 0.f);
    return cdf > 0.f || h != h ? h * cdf : 0.f;
  }
  if (act == ATOMO_ACT_SILU) {
    const float s = 1.f / (1.f + expf(-h));
    // where s is 0 its product with h is, too, and not 0 * -inf
    const float y = s > 0.f || h != h ? h * s : 0.f;
    *slope = s + (s < 1.f ? y * (1.f - s) : 0.f);
    return y;
  }
  *slope = 1.f;
  return h;
}

constexpr int kRowBytes = 128;  // of the reduction, in a tile
constexpr int kRowChunks = kRowBytes / 16;

// Where chunk c of a tile's row lies: eight neighbouring rows (a fragment's
// read) and eight rows four apart (a transposed block's write) both fall on
// eight different chunks, that is, on all banks.
__device__ __forceinline__ int slot(int row, int c) {
  return row * kRowChunks + (c ^ ((row ^ (row >> 3)) & 7));
}

// Tile of kRows rows by kRowBytes of the reduction, from memory to LDS.
template <typename E, int kRows, int kThreads, bool kAcross>
struct Stage {
  using Raw = typename E::Raw;
  static constexpr int kC = E::kChunk;
  static constexpr int kK = kRowBytes / sizeof(Raw);
  static constexpr int kVecs = kRows * kRowChunks / kThreads;
  u32x4 v[kVecs];

  // `at` points at row 0, reduction 0 of the tile; rows and ks remain there
  __device__ __forceinline__ void load(const Raw* at, int64_t ld, int rows,
                                       int ks) {
    if constexpr (!kAcross) {
#pragma unroll
      for (int s = 0; s < kVecs; ++s) {
        const int id = threadIdx.x + s * kThreads;
        const int row = id / kRowChunks, k = id % kRowChunks * kC;
        u32x4 r = {0, 0, 0, 0};
        if (row < rows && k < ks) {
          const Raw* src = at + row * ld + k;
          if (k + kC <= ks) {
            if constexpr (sizeof(Raw) == 4)
              r = *(const u32x4_a4*)src;
            else
              r = *(const u32x4_a2*)src;
          } else {
#pragma unroll
            for (int e = 0; e < kC; ++e) {
              if (k + e < ks) {
                if constexpr (sizeof(Raw) == 4)
                  r[e] = src[e];
                else
                  r[e / 2] |= (uint32_t)src[e] << (e % 2 * 16);
              }
            }
          }
        }
        v[s] = r;
      }
    } else {
      // blocks of kC k by 4 rows; neighbouring threads take neighbouring rows
      constexpr int kBlocks = kRows / 4 * kRowChunks / kThreads;
      static_assert(kBlocks * 4 == kVecs, "a block is four chunks");
#pragma unroll
      for (int b = 0; b < kBlocks; ++b) {
        const int id = threadIdx.x + b * kThreads;
        const int row = id % (kRows / 4) * 4, k = id / (kRows / 4) * kC;
        if constexpr (sizeof(Raw) == 4) {
          u32x4 in[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            u32x4 r = {0, 0, 0, 0};
            if (k + e < ks && row < rows) {
              const Raw* src = at + (k + e) * ld + row;
              if (row + 4 <= rows) {
                r = *(const u32x4_a4*)src;
              } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                  if (row + i < rows) r[i] = src[i];
              }
            }
            in[e] = r;
          }
#pragma unroll
          for (int i = 0; i < 4; ++i)
            v[b * 4 + i] = u32x4{in[0][i], in[1][i], in[2][i], in[3][i]};
        } else {
          u32x2 in[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            u32x2 r = {0, 0};
            if (k + e < ks && row < rows) {
              const Raw* src = at + (k + e) * ld + row;
              if (row + 4 <= rows) {
                r = *(const u32x2_a2*)src;
              } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                  if (row + i < rows)
                    r[i / 2] |= (uint32_t)src[i] << (i % 2 * 16);
              }
            }
            in[e] = r;
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            // the low or the high halves of two k
            const uint32_t pick = i % 2 ? 0x07060302u : 0x05040100u;
#pragma unroll
            for (int e = 0; e < 4; ++e)
              v[b * 4 + i][e] = __builtin_amdgcn_perm(
                  in[2 * e + 1][i / 2], in[2 * e][i / 2], pick);
          }
        }
      }
    }
  }

  __device__ __forceinline__ void store(u32x4* tile) const {
    if constexpr (!kAcross) {
#pragma unroll
      for (int s = 0; s < kVecs; ++s) {
        const int id = threadIdx.x + s * kThreads;
        tile[slot(id / kRowChunks, id % kRowChunks)] = v[s];
      }
    } else {
#pragma unroll
      for (int s = 0; s < kVecs; ++s) {
        const int id = threadIdx.x + s / 4 * kThreads;
        tile[slot(id % (kRows / 4) * 4 + s % 4, id / (kRows / 4))] = v[s];
      }
    }
  }
};

constexpr int kTile = 128;
constexpr int kThreads = 256;

// 128 x 128 of the result by 4 waves of 64 x 64 each, tiles of 128 bytes of
// the reduction, double-buffered in LDS (64 KB: two workgroups a CU).
template <typename E, bool kAcrossP, bool kAcrossQ>
__global__ void __launch_bounds__(kThreads)
    product_kernel(AtomoProduct a, int tiles_i, int tiles_j) {
  using Raw = typename E::Raw;
  __shared__ u32x4 lds[2][2][kTile * kRowChunks];
  constexpr int kK = kRowBytes / sizeof(Raw);
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  const int i0 = blockIdx.x % tiles_i * kTile;
  const int j0 = blockIdx.x / tiles_i * kTile;
  const int rows_i = min(a.ni - i0, kTile), rows_j = min(a.nj - j0, kTile);
  const Raw* p = (const Raw*)a.p + (kAcrossP ? (int64_t)i0 : i0 * a.ldp);
  const Raw* q = (const Raw*)a.q + (kAcrossQ ? (int64_t)j0 : j0 * a.ldq);
  const int64_t step_p = kAcrossP ? a.ldp * kK : kK;
  const int64_t step_q = kAcrossQ ? a.ldq * kK : kK;
  const int steps = (a.nk + kK - 1) / kK;

  f32x16 acc[2][2] = {};
  Stage<E, kTile, kThreads, kAcrossP> sp;
  Stage<E, kTile, kThreads, kAcrossQ> sq;
  sp.load(p, a.ldp, rows_i, a.nk);
  sq.load(q, a.ldq, rows_j, a.nk);
  sp.store(lds[0][0]);
  sq.store(lds[0][1]);
  __syncthreads();
  const int wi = wave % 2 * 64 + lane % 32, wj = wave / 2 * 64 + lane % 32;
  for (int s = 0; s < steps; ++s) {
    const bool more = s + 1 < steps;
    if (more) {
      sp.load(p + (s + 1) * step_p, a.ldp, rows_i, a.nk - (s + 1) * kK);
      sq.load(q + (s + 1) * step_q, a.ldq, rows_j, a.nk - (s + 1) * kK);
    }
    const u32x4* tp = lds[s & 1][0];
    const u32x4* tq = lds[s & 1][1];
#pragma unroll
    for (int c = 0; c < kRowChunks; c += 2) {
      u32x4 fp[2], fq[2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        fp[t] = tp[slot(wi + t * 32, c + lane / 32)];
        fq[t] = tq[slot(wj + t * 32, c + lane / 32)];
      }
#pragma unroll
      for (int ti = 0; ti < 2; ++ti)
#pragma unroll
        for (int tj = 0; tj < 2; ++tj) multiply<E>(fp[ti], fq[tj], acc[ti][tj]);
    }
    if (more) {
      sp.store(lds[(s + 1) & 1][0]);
      sq.store(lds[(s + 1) & 1][1]);
    }
    __syncthreads();
  }

  // a lane holds i = 8 g + 4 (lane / 32) + 0..3 of j = lane % 32
  const Raw* bias = (const Raw*)a.bias;
#pragma unroll
  for (int ti = 0; ti < 2; ++ti)
#pragma unroll
    for (int tj = 0; tj < 2; ++tj) {
      const int j = j0 + wj + tj * 32;
      if (j >= a.nj) continue;
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int i = i0 + wave % 2 * 64 + ti * 32 + g * 8 + lane / 32 * 4;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (i + e >= a.ni) break;
          float h = acc[ti][tj][g * 4 + e];
          if (bias) h += E::widen(bias[i + e]);
          float slope;
          float y = activate(a.act, h, &slope);
          if (a.slope)
            ((Raw*)a.slope)[(int64_t)j * a.ni + i + e] = E::narrow(slope);
          if (a.residual)
            y += E::widen(((const Raw*)a.residual)[j * a.ldr + i + e]);
          ((Raw*)a.out)[j * a.ldo + i + e] = E::narrow(y);
        }
      }
    }
}

// dp and the partial column sums of a block of rows; a thread a column
template <typename E>
__global__ void __launch_bounds__(kThreads)
    linear_dp_kernel(const typename E::Raw* __restrict__ dy, int64_t ld_dy,
                     const typename E::Raw* __restrict__ slope, int by_output,
                     typename E::Raw* __restrict__ dp,
                     float* __restrict__ partial, int rows, int columns,
                     int block_rows) {
  const int c = blockIdx.x * kThreads + threadIdx.x;
  if (c >= columns) return;
  const int first = blockIdx.y * block_rows;
  const int last = min(rows, first + block_rows);
  float sum = 0.f;
  for (int r = first; r < last; ++r) {
    float d = E::widen(dy[r * ld_dy + c]);
    if (slope) {
      const float s = E::widen(slope[(int64_t)r * columns + c]);
      if (by_output)
        d = s <= 0.f ? 0.f : d;
      else
        d *= s;
    }
    const typename E::Raw raw = E::narrow(d);
    if (dp) dp[(int64_t)r * columns + c] = raw;
    sum += d;
  }
  if (partial) partial[(int64_t)blockIdx.y * columns + c] = sum;
}

template <typename E>
__global__ void __launch_bounds__(kThreads)
    linear_db_kernel(const float* __restrict__ partial, int blocks, int columns,
                     typename E::Raw* __restrict__ db) {
  const int c = blockIdx.x * kThreads + threadIdx.x;
  if (c >= columns) return;
  float sum = 0.f;
  for (int b = 0; b < blocks; ++b) sum += partial[(int64_t)b * columns + c];
  db[c] = E::narrow(sum);
}

template <typename E>
void product(const AtomoProduct& a, hipStream_t stream) {
  const int ti = (a.ni + kTile - 1) / kTile, tj = (a.nj + kTile - 1) / kTile;
  const dim3 grid(ti * tj), block(kThreads);
  if (a.form == ATOMO_FORWARD)
    hipLaunchKernelGGL((product_kernel<E, false, false>), grid, block, 0,
                       stream, a, ti, tj);
  else if (a.form == ATOMO_GRAD_X)
    hipLaunchKernelGGL((product_kernel<E, true, false>), grid, block, 0, stream,
                       a, ti, tj);
  else
    hipLaunchKernelGGL((product_kernel<E, true, true>), grid, block, 0, stream,
                       a, ti, tj);
}

template <typename E>
void linear_dp(const void* dy, int64_t ld_dy, const void* slope, int by_output,
               void* dp, void* db, float* partial, int row_blocks, int rows,
               int columns, hipStream_t stream) {
  using Raw = typename E::Raw;
  const int wide = (columns + kThreads - 1) / kThreads;
  hipLaunchKernelGGL((linear_dp_kernel<E>), dim3(wide, row_blocks),
                     dim3(kThreads), 0, stream, (const Raw*)dy, ld_dy,
                     (const Raw*)slope, by_output, (Raw*)dp,
                     db ? partial : nullptr, rows, columns,
                     (rows + row_blocks - 1) / row_blocks);
  if (db)
    hipLaunchKernelGGL((linear_db_kernel<E>), dim3(wide), dim3(kThreads), 0,
                       stream, partial, row_blocks, columns, (Raw*)db);
}

}  // namespace

extern "C" {

void atomo_product_launch(const AtomoProduct* a, hipStream_t stream) {
  if (a->type == ATOMO_F32)
    product<F32>(*a, stream);
  else if (a->type == ATOMO_BF16)
    product<BF16>(*a, stream);
  else
    product<F16>(*a, stream);
}

void atomo_linear_dp_launch(const void* dy, int64_t ld_dy, const void* slope,
                            int by_output, void* dp, void* db, float* partial,
                            int row_blocks, int rows, int columns, int type,
                            hipStream_t stream) {
  if (type == ATOMO_F32)
    linear_dp<F32>(dy, ld_dy, slope, by_output, dp, db, partial, row_blocks,
                   rows, columns, stream);
  else if (type == ATOMO_BF16)
    linear_dp<BF16>(dy, ld_dy, slope, by_output, dp, db, partial, row_blocks,
                    rows, columns, stream);
  else
    linear_dp<F16>(dy, ld_dy, slope, by_output, dp, db, partial, row_blocks,
                   rows, columns, stream);
}

}  // extern "C"
