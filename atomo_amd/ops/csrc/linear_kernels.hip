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
// neighbouring k each).  Aligned 16-bit operands go to LDS directly, as they
// lie, and are transposed as they are read (product_direct_kernel).  p gives the rows of the matrix instruction's result:
// a lane then holds four neighbouring i of one j, and stores them at once.
//
// Sums are fp32; an output is rounded once.
//
// Sizes decide the tile and in how many parts the reduction is made
// (atomo_product_plan); few rows have a kernel of their own.

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
  static constexpr Raw kMinusZero = 0x80000000u;
  static constexpr int kChunk = 4;  // elements in 16 bytes
  __device__ static float widen(Raw r) { return __uint_as_float(r); }
  __device__ static Raw narrow(float f) { return __float_as_uint(f); }
};
struct BF16 {
  using Raw = uint16_t;
  static constexpr Raw kMinusZero = 0x8000u;
  static constexpr int kChunk = 8;
  __device__ static float widen(Raw r) {
    return __uint_as_float((uint32_t)r << 16);
  }
  __device__ static Raw narrow(float f) {
    return __builtin_bit_cast(Raw, (__bf16)f);
  }
  __device__ static f32x16 multiply(const u32x4& p, const u32x4& q, f32x16 acc) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(
        __builtin_bit_cast(bf16x8, p), __builtin_bit_cast(bf16x8, q), acc, 0, 0,
        0);
  }
};
struct F16 {
  using Raw = uint16_t;
  static constexpr Raw kMinusZero = 0x8000u;
  static constexpr int kChunk = 8;
  __device__ static float widen(Raw r) {
    return (float)__builtin_bit_cast(_Float16, r);
  }
  __device__ static Raw narrow(float f) {
    return __builtin_bit_cast(Raw, (_Float16)f);
  }
  __device__ static f32x16 multiply(const u32x4& p, const u32x4& q, f32x16 acc) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(
        __builtin_bit_cast(f16x8, p), __builtin_bit_cast(f16x8, q), acc, 0, 0,
        0);
  }
};

// acc[i][j] += the products of 16 bytes of p's rows i and q's rows j
template <typename E, int kI, int kJ>
__device__ __forceinline__ void multiply(const u32x4 (&p)[kI],
                                         const u32x4 (&q)[kJ],
                                         f32x16 (&acc)[kI][kJ]) {
  if constexpr (E::kChunk == 4) {
    // neighbouring instructions add to different tiles: none waits
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
      for (int i = 0; i < kI; ++i)
#pragma unroll
        for (int j = 0; j < kJ; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x2f32(
              __uint_as_float(p[i][c]), __uint_as_float(q[j][c]), acc[i][j], 0,
              0, 0);
  } else {
#pragma unroll
    for (int i = 0; i < kI; ++i)
#pragma unroll
      for (int j = 0; j < kJ; ++j) acc[i][j] = E::multiply(p[i], q[j], acc[i][j]);
  }
}

// Half the complementary error function of -h / sqrt(2), and exp(-h^2 / 2).
// Beside 16-bit results by their quotient, which varies slowly: a polynomial
// in t = 1 / (1 + 0.36 |h|), fitted so that its largest relative error over
// h = -13.5..0 is least, 2^-20; the exponential's exponent, rounded twice, adds
// h^2 2^-24.  So a result is within 2^-17 of itself down to h = -8 and rounded
// once.  It costs nothing that can be measured against a polynomial that is
// good in absolute terms only: 8192 x 4096 x 4096 bf16 with gelu, forward and
// backward, 801 us with either.
template <bool kShort>
__device__ __forceinline__ float normal_cdf(float h, float* bell) {
  if constexpr (kShort) {
    const float t = __builtin_amdgcn_rcpf(1.f + 0.36f * fabsf(h));
    const float e = __builtin_amdgcn_exp2f(h * h * -0.72134752044448170f);
    const float p =
        ((((((0.047306422f * t - 0.18061617f) * t + 0.18210846f) * t +
            0.025755247f) * t + 0.14001004f) * t + 0.14171898f) * t +
         0.14371689f) * t * e;
    *bell = e;
    return h < 0.f ? p : 1.f - p;
  } else {
    *bell = expf(-0.5f * h * h);
    return 0.5f * erfcf(h * -0.70710678118654752f);
  }
}

// y and dy/dh of the activation at h
template <bool kShort>
__device__ __forceinline__ float activate(int act, float h, float* slope) {
  if (act == ATOMO_ACT_RELU) {
    // not (h <= 0): NaN passes
    *slope = h <= 0.f ? 0.f : 1.f;
    return h <= 0.f ? 0.f : h;
  }
  if (act == ATOMO_ACT_GELU) {
    float bell;
    const float cdf = normal_cdf<kShort>(h, &bell);
    // beyond the bell both are what they tend to, not 0 * inf
    *slope = cdf + (bell > 0.f ? h * bell * 0.39894228040143268f : 0.f);
    return cdf > 0.f || h != h ? h * cdf : 0.f;
  }
  if (act == ATOMO_ACT_SILU) {
    const float e = __builtin_amdgcn_exp2f(h * -1.44269504088896341f);
    const float s = kShort ? __builtin_amdgcn_rcpf(1.f + e) : 1.f / (1.f + e);
    // where s is 0 its product with h is, too, and not 0 * -inf
    const float y = s > 0.f || h != h ? h * s : 0.f;
    *slope = s + (s < 1.f ? y * (1.f - s) : 0.f);
    return y;
  }
  *slope = 1.f;
  return h;
}

// An output from its fp32 value.  Of relu without a residual the backward pass
// reads the slope off the output: a value above 0 that the type rounds to 0
// (fp16: below 2^-25) is written as -0, which is equal to 0, and is not lost.
template <typename E>
__device__ __forceinline__ typename E::Raw output(const AtomoProduct& a, float y) {
  const typename E::Raw r = E::narrow(y);
  const bool lost = a.act == ATOMO_ACT_RELU && !a.residual && y > 0.f && r == 0;
  return lost ? E::kMinusZero : r;
}
template <typename E>
__device__ __forceinline__ bool relu_is_off(typename E::Raw y) {
  return E::widen(y) <= 0.f && y != E::kMinusZero;
}

constexpr int kRowBytes = 128;  // of the reduction, in a tile
constexpr int kRowChunks = kRowBytes / 16;

// Where chunk c of a tile's row lies: eight neighbouring rows (a fragment's
// read) and eight rows four apart (a transposed block's write) both fall on
// eight different chunks, that is, on all banks.
__device__ __forceinline__ int slot(int row, int c) {
  return row * kRowChunks + (c ^ ((row ^ (row >> 3)) & 7));
}

// A row of a bf16 plane of an fp32 tile: 32 elements, four chunks.  Eight
// neighbouring rows, and sixteen, fall on different banks.
constexpr int kThirdBytes = 64;
__device__ __forceinline__ int third_slot(int row, int c) {
  return row * 4 + (c ^ ((row >> 1) & 3) ^ ((row >> 3) & 3));
}

// Elements 4 c4 .. 4 c4 + 3 of a row as x = a + b + c: a the bf16 next to x, b
// the one next to x - a, c the rest: 3 x 8 bits hold the 24 of an fp32.
__device__ __forceinline__ void put_thirds(char* tile, int plane, int row, int c4,
                                           const u32x4& x) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  char* to = tile + third_slot(row, c4 / 2) * 16 + c4 % 2 * 8;
  float r[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) r[e] = __uint_as_float(x[e]);
#pragma unroll
  for (int t = 0; t < 3; ++t) {
    u32x2 out;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const bf16x2 near = {(__bf16)r[2 * h], (__bf16)r[2 * h + 1]};
      out[h] = __builtin_bit_cast(uint32_t, near);
      r[2 * h] -= __uint_as_float(out[h] << 16);
      r[2 * h + 1] -= __uint_as_float(out[h] & 0xFFFF0000u);
    }
    *(u32x2*)(to + t * plane) = out;
  }
}

// Tile of kRows rows by kRowBytes of the reduction, from memory to LDS.  What
// is loaded is not touched before store(), so that nothing waits for it.
template <typename E, int kRows, int kThreads, bool kAcross>
struct Stage {
  using Raw = typename E::Raw;
  static constexpr int kC = E::kChunk;
  // An operand that lies across is taken in blocks of kC k by 4 rows;
  // neighbouring threads take neighbouring rows.
  static constexpr int kAll = kRows / 4 * kRowChunks;
  static constexpr int kBlocks = (kAll + kThreads - 1) / kThreads;
  static constexpr int kVecs =
      kAcross ? kBlocks * 4 : kRows * kRowChunks / kThreads;
  u32x4 v[kVecs];  // across, 16-bit: v[..][2 (k % 2)..] holds four rows of a k

  __device__ static bool idle(int id) {
    return kAll % kThreads != 0 && id >= kAll;
  }

  // All of it lies in memory, but for rows from `rows` on: others are read in
  // their place, or, where it lies across, up to three elements that follow;
  // both only reach results that nobody keeps.
  __device__ __forceinline__ void load_whole(const Raw* at, int64_t ld,
                                             int rows) {
    if constexpr (!kAcross) {
#pragma unroll
      for (int s = 0; s < kVecs; ++s) {
        const int id = threadIdx.x + s * kThreads;
        const Raw* src = at + min(id / kRowChunks, rows - 1) * ld +
                         id % kRowChunks * kC;
        if constexpr (kC == 4)
          v[s] = *(const u32x4_a4*)src;
        else
          v[s] = *(const u32x4_a2*)src;
      }
    } else {
#pragma unroll
      for (int b = 0; b < kBlocks; ++b) {
        const int id = threadIdx.x + b * kThreads;
        if (idle(id)) break;
        const Raw* src = at + (int64_t)(id / (kRows / 4) * kC) * ld +
                         min(id % (kRows / 4) * 4, (rows - 1) & ~3);
#pragma unroll
        for (int e = 0; e < kC; ++e) {
          if constexpr (kC == 4) {
            v[b * 4 + e] = *(const u32x4_a4*)(src + e * ld);
          } else {
            const u32x2 r = *(const u32x2_a2*)(src + e * ld);
            v[b * 4 + e / 2][e % 2 * 2] = r[0];
            v[b * 4 + e / 2][e % 2 * 2 + 1] = r[1];
          }
        }
      }
    }
  }

  // `at` points at row 0, reduction 0 of the tile; rows and ks remain there,
  // zeros follow in the reduction.  A vector that would pass an end is read
  // up to that end and moved into place, so the matrix has to hold a vector.
  __device__ __forceinline__ void load_edge(const Raw* at, int64_t ld, int rows,
                                            int ks) {
    if constexpr (!kAcross) {
#pragma unroll
      for (int s = 0; s < kVecs; ++s) {
        const int id = threadIdx.x + s * kThreads;
        const int k = id % kRowChunks * kC, from = min(k, ks - kC);
        const Raw* src = at + min(id / kRowChunks, rows - 1) * ld + from;
        u32x4 r;
        if constexpr (kC == 4)
          r = *(const u32x4_a4*)src;
        else
          r = *(const u32x4_a2*)src;
        // down by what an earlier vector holds as well, zeros after it
        const int by = k - from;
        if constexpr (kC == 4) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            uint32_t x = by == 0 ? r[e] : 0;
#pragma unroll
            for (int d = 1; d < 4 - e; ++d) x = by == d ? r[e + d] : x;
            r[e] = x;
          }
        } else {
          uint64_t lo = ((uint64_t)r[1] << 32) | r[0];
          uint64_t hi = ((uint64_t)r[3] << 32) | r[2];
          if (by >= 4) {
            lo = by < 8 ? hi >> (by * 16 - 64) : 0;
            hi = 0;
          } else if (by > 0) {
            lo = lo >> (by * 16) | hi << (64 - by * 16);
            hi >>= by * 16;
          }
          r = u32x4{(uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi,
                    (uint32_t)(hi >> 32)};
        }
        v[s] = r;
      }
    } else {
#pragma unroll
      for (int b = 0; b < kBlocks; ++b) {
        const int id = threadIdx.x + b * kThreads;
        if (idle(id)) break;
        const int k = id / (kRows / 4) * kC;
        const int row = min(id % (kRows / 4) * 4, rows - 1);
        const int from = min(row, rows - 4), by = row - from;
#pragma unroll
        for (int e = 0; e < kC; ++e) {
          const Raw* src = at + (int64_t)min(k + e, ks - 1) * ld + from;
          const bool there = k + e < ks;
          if constexpr (kC == 4) {
            const u32x4 r = *(const u32x4_a4*)src;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              uint32_t x = r[i];
#pragma unroll
              for (int d = 1; d < 4 - i; ++d) x = by == d ? r[i + d] : x;
              v[b * 4 + e][i] = there ? x : 0;
            }
          } else {
            const u32x2 r = *(const u32x2_a2*)src;
            const uint64_t x = there ? (((uint64_t)r[1] << 32) | r[0]) >> (by * 16)
                                     : 0;
            v[b * 4 + e / 2][e % 2 * 2] = (uint32_t)x;
            v[b * 4 + e / 2][e % 2 * 2 + 1] = (uint32_t)(x >> 32);
          }
        }
      }
    }
  }

  // Element by element, for matrices that hold no vector.
  __device__ __forceinline__ void load_tiny(const Raw* at, int64_t ld, int rows,
                                            int ks) {
#pragma unroll
    for (int s = 0; s < kVecs; ++s) v[s] = u32x4{0, 0, 0, 0};
    if constexpr (!kAcross) {
#pragma unroll
      for (int s = 0; s < kVecs; ++s) {
        const int id = threadIdx.x + s * kThreads;
        const int row = id / kRowChunks, k = id % kRowChunks * kC;
        if (row >= rows) continue;
        const Raw* src = at + row * ld + k;
#pragma unroll
        for (int e = 0; e < kC; ++e) {
          if (k + e >= ks) continue;
          if constexpr (kC == 4)
            v[s][e] = src[e];
          else
            v[s][e / 2] |= (uint32_t)src[e] << (e % 2 * 16);
        }
      }
    } else {
#pragma unroll
      for (int b = 0; b < kBlocks; ++b) {
        const int id = threadIdx.x + b * kThreads;
        if (idle(id)) break;
        const int row = id % (kRows / 4) * 4, k = id / (kRows / 4) * kC;
#pragma unroll
        for (int e = 0; e < kC; ++e) {
          if (k + e >= ks) continue;
          const Raw* src = at + (k + e) * ld + row;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (row + i >= rows) continue;
            if constexpr (kC == 4)
              v[b * 4 + e][i] = src[i];
            else
              v[b * 4 + e / 2][e % 2 * 2 + i / 2] |= (uint32_t)src[i]
                                                     << (i % 2 * 16);
          }
        }
      }
    }
  }

  // fp32 as three bf16 planes, `plane` bytes apart
  __device__ __forceinline__ void store_thirds(char* tile, int plane) const {
    static_assert(kC == 4, "fp32");
    if constexpr (!kAcross) {
#pragma unroll
      for (int s = 0; s < kVecs; ++s) {
        const int id = threadIdx.x + s * kThreads;
        put_thirds(tile, plane, id / kRowChunks, id % kRowChunks, v[s]);
      }
    } else {
#pragma unroll
      for (int b = 0; b < kBlocks; ++b) {
        const int id = threadIdx.x + b * kThreads;
        if (idle(id)) break;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          put_thirds(tile, plane, id % (kRows / 4) * 4 + i, id / (kRows / 4),
                     u32x4{v[b * 4][i], v[b * 4 + 1][i], v[b * 4 + 2][i],
                           v[b * 4 + 3][i]});
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
      for (int b = 0; b < kBlocks; ++b) {
        const int id = threadIdx.x + b * kThreads;
        if (idle(id)) break;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          u32x4 out;
          // the low or the high halves of two k
          const uint32_t pick = i % 2 ? 0x07060302u : 0x05040100u;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if constexpr (kC == 4)
              out[e] = v[b * 4 + e][i];
            else
              out[e] = __builtin_amdgcn_perm(v[b * 4 + e][2 + i / 2],
                                             v[b * 4 + e][i / 2], pick);
          }
          tile[slot(id % (kRows / 4) * 4 + i, id / (kRows / 4))] = out;
        }
      }
    }
  }
};

// neighbours in a row, at the alignment of one
template <typename Raw, int kN>
struct Some {
  Raw v[kN];
} __attribute__((packed, aligned(sizeof(Raw))));
template <typename Raw>
using Four = Some<Raw, 4>;

// the first n of them
template <int kN, typename Raw>
__device__ __forceinline__ Some<Raw, kN> load_some(const Raw* at, int n) {
  Some<Raw, kN> f = {};
  if (n >= kN) return *(const Some<Raw, kN>*)at;
#pragma unroll
  for (int e = 0; e < kN - 1; ++e)
    if (e < n) f.v[e] = at[e];
  return f;
}
template <int kN, typename Raw>
__device__ __forceinline__ void store_some(Raw* at, int n,
                                           const Some<Raw, kN>& f) {
  if (n >= kN) {
    *(Some<Raw, kN>*)at = f;
    return;
  }
#pragma unroll
  for (int e = 0; e < kN - 1; ++e)
    if (e < n) at[e] = f.v[e];
}

// Bias, activation, residual and slope on four neighbouring sums of row j, of
// which the columns below a.ni exist.
template <typename E>
__device__ __forceinline__ void finish(const AtomoProduct& a, int64_t j, int i,
                                       const float (&sum)[4],
                                       const Four<typename E::Raw>& bias,
                                       const Four<typename E::Raw>& residual) {
  using Raw = typename E::Raw;
  Four<Raw> y;
  // fp32, whatever the operands: the slopes of gelu and silu fall to 0 without
  // an end, and next to their zero they need digits that 16 bits do not have.
  // (8192 x 4096 bf16: 67 MB more here and in linear_dp_kernel.)
  Four<float> s;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    float h = sum[e], d;
    if (a.bias) h += E::widen(bias.v[e]);
    h = activate<E::kChunk == 8>(a.act, h, &d);
    s.v[e] = d;
    if (a.residual) h += E::widen(residual.v[e]);
    y.v[e] = output<E>(a, h);
  }
  store_some<4>((Raw*)a.out + j * a.ldo + i, a.ni - i, y);
  if (a.slope) store_some<4>((float*)a.slope + j * a.ni + i, a.ni - i, s);
}

template <typename E>
__device__ __forceinline__ Four<typename E::Raw> bias_of(const AtomoProduct& a,
                                                         int i) {
  if (!a.bias || i >= a.ni) return {};
  return load_some<4>((const typename E::Raw*)a.bias + i, a.ni - i);
}
template <typename E>
__device__ __forceinline__ Four<typename E::Raw> residual_of(
    const AtomoProduct& a, int64_t j, int i) {
  if (!a.residual || i >= a.ni || j >= a.nj) return {};
  return load_some<4>((const typename E::Raw*)a.residual + j * a.ldr + i, a.ni - i);
}

// lanes of one wave read in LDS what others of it wrote
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Which part of a product a workgroup makes.
template <typename E, bool kAcrossP, bool kAcrossQ, int kI, int kJ>
struct Work {
  using Raw = typename E::Raw;
  static constexpr int kK = kRowBytes / sizeof(Raw);  // a step's reduction
  int part, i0, j0, rows_i, rows_j, ks, steps, whole, begin;
  const Raw *p, *q;

  __device__ explicit Work(const AtomoProduct& a) {
    // Workgroups go round the 8 XCDs: each is given neighbouring tiles, in
    // bands of kBand, so that its L2 holds what they share (8192 x 4096 x 4096
    // bf16: 398 -> 375 us).
    constexpr int kXcds = 8, kBand = 4;
    const int tiles_i = (a.ni + kI - 1) / kI, tiles_j = (a.nj + kJ - 1) / kJ;
    const int tiles = tiles_i * tiles_j, all = tiles * a.splits;
    const int xcd = blockIdx.x % kXcds;
    const int at = xcd * (all / kXcds) + min(xcd, all % kXcds) +
                   (int)(blockIdx.x / kXcds);
    const int tile = at % tiles;
    const int band = tile / (kBand * tiles_i), in = tile % (kBand * tiles_i);
    const int band_j = min(kBand, tiles_j - band * kBand);
    const int tile_i = in / band_j, tile_j = band * kBand + in % band_j;
    part = at / tiles;
    i0 = tile_i * kI;
    j0 = tile_j * kJ;
    rows_i = min(a.ni - i0, kI);
    rows_j = min(a.nj - j0, kJ);
    const int k0 = part * a.k_part;
    ks = min(a.nk - k0, a.k_part);
    steps = (ks + kK - 1) / kK;
    p = (const Raw*)a.p + (kAcrossP ? (int64_t)k0 * a.ldp + i0 : i0 * a.ldp + k0);
    q = (const Raw*)a.q + (kAcrossQ ? (int64_t)k0 * a.ldq + j0 : j0 * a.ldq + k0);
    // Steps that load_whole() may take.  Blocks of four that pass the end of
    // their row end in the next one: there has to be one.
    const bool past_p = kAcrossP && rows_i % 4, past_q = kAcrossQ && rows_j % 4;
    const bool next = !((past_p && a.ldp < 3) || (past_q && a.ldq < 3));
    const int last = past_p || past_q ? min(ks, a.nk - 1 - k0) : ks;
    whole = next ? last / kK : 0;
    // Neighbours start at different steps: rows of a power of two bytes put
    // all that one step reads on a few of L2's channels (dW of 8192 x 4096 x
    // 4096 bf16: 619 -> 322 us).  The order of the sum depends on the tile
    // alone.
    begin = (tile_i + tile_j) % 16 * 2 % steps;
  }

  template <bool kTiny, typename P, typename Q>
  __device__ __forceinline__ void load(const AtomoProduct& a, int s, P& sp,
                                       Q& sq) const {
    s += begin;
    s = s < steps ? s : s - steps;
    const Raw* at_p = p + s * (kAcrossP ? a.ldp * kK : (int64_t)kK);
    const Raw* at_q = q + s * (kAcrossQ ? a.ldq * kK : (int64_t)kK);
    if constexpr (kTiny) {
      sp.load_tiny(at_p, a.ldp, rows_i, ks - s * kK);
      sq.load_tiny(at_q, a.ldq, rows_j, ks - s * kK);
    } else if (s < whole) {
      sp.load_whole(at_p, a.ldp, rows_i);
      sq.load_whole(at_q, a.ldq, rows_j);
    } else {
      sp.load_edge(at_p, a.ldp, rows_i, ks - s * kK);
      sq.load_edge(at_q, a.ldq, rows_j, ks - s * kK);
    }
  }
};

// Four neighbouring sums without an epilogue, or of a part of the reduction.
template <typename E>
__device__ __forceinline__ void put_bare(const AtomoProduct& a, int part,
                                         int64_t j, int i, const float4& v) {
  using Raw = typename E::Raw;
  if (i >= a.ni) return;
  if (a.splits > 1) {
    // rows of a multiple of four: whole vectors
    *(float4*)(a.partial + ((int64_t)part * a.nj + j) * a.ld_part + i) = v;
    return;
  }
  const Four<Raw> y = {{E::narrow(v.x), E::narrow(v.y), E::narrow(v.z),
                        E::narrow(v.w)}};
  store_some<4>((Raw*)a.out + j * a.ldo + i, a.ni - i, y);
}

// A wave's sums, from row i0 and column j0 of the result on, to the epilogue
// or to `partial`.  A lane holds i = 8 g + 4 (lane / 32) + 0..3 of j =
// lane % 32.  By way of LDS (`mine`, the wave's own part, rows padded by 16
// bytes against the banks) it gets four neighbours of a row of kPass, so that
// lines are written whole and the epilogue's code is a short loop.
template <int kFi>
constexpr int pass_floats() {
  return 32 * ((kFi > 1 ? 64 : 32) + 4);
}

template <typename E, int kFi, int kFj>
__device__ __forceinline__ void write_tile(const AtomoProduct& a, int part,
                                           int i0, int64_t j0,
                                           const f32x16 (&acc)[kFi][kFj],
                                           float* mine) {
  constexpr int kPass = kFi > 1 ? 64 : 32, kPitch = kPass + 4;
  constexpr int kLanes = kPass / 4;  // of a row
  const int lane = threadIdx.x % 64;
#pragma unroll
  for (int ti = 0; ti < kFi; ti += kPass / 32)
#pragma unroll
    for (int tj = 0; tj < kFj; ++tj) {
#pragma unroll
      for (int t = 0; t < kPass / 32; ++t)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          *(float4*)(mine + lane % 32 * kPitch + t * 32 + g * 8 + lane / 32 * 4) =
              make_float4(acc[ti + t][tj][g * 4], acc[ti + t][tj][g * 4 + 1],
                          acc[ti + t][tj][g * 4 + 2], acc[ti + t][tj][g * 4 + 3]);
      wave_sync();
      constexpr int kRows = 64 / kLanes;  // of the pass, at a time
      const int i = i0 + ti * 32 + lane % kLanes * 4;
      const int64_t j = j0 + tj * 32 + lane / kLanes;
      const float* from = mine + lane / kLanes * kPitch + lane % kLanes * 4;
      if (a.bare) {
        // nothing but stores: all reads go before the first
        float4 v[32 / kRows];
#pragma unroll
        for (int r = 0; r < 32 / kRows; ++r)
          v[r] = *(const float4*)(from + r * kRows * kPitch);
#pragma unroll
        for (int r = 0; r < 32 / kRows; ++r)
          if (j + r * kRows < a.nj) put_bare<E>(a, part, j + r * kRows, i, v[r]);
      } else {
        // all that four rows need is read before the first is worked on
        constexpr int kBatch = 32 / kRows < 4 ? 32 / kRows : 4;
        const Four<typename E::Raw> bias = bias_of<E>(a, i);
#pragma unroll 1
        for (int r0 = 0; r0 < 32; r0 += kRows * kBatch) {
          float4 v[kBatch];
          Four<typename E::Raw> residual[kBatch];
          const auto load = [&](int n) {
#pragma unroll
            for (int r = 0; r < kBatch; ++r)
              residual[r] = load_some<4>(
                  (const typename E::Raw*)a.residual +
                      min(j + r0 + r * kRows, (int64_t)a.nj - 1) * a.ldr + i,
                  n);
          };
          // whole ones apart, without a branch in between
          if (a.residual && i + 4 <= a.ni)
            load(4);
          else if (a.residual && i < a.ni)
            load(a.ni - i);
#pragma unroll
          for (int r = 0; r < kBatch; ++r)
            v[r] = *(const float4*)(from + (r0 + r * kRows) * kPitch);
#pragma unroll
          for (int r = 0; r < kBatch; ++r) {
            const int64_t jr = j + r0 + r * kRows;
            const float sum[4] = {v[r].x, v[r].y, v[r].z, v[r].w};
            if (jr < a.nj && i < a.ni)
              finish<E>(a, jr, i, sum, bias, residual[r]);
          }
        }
      }
      wave_sync();
    }
}

// kI x kJ of the result by kWi x kWj waves; a tile of the reduction is 128
// bytes of each row, double-buffered in LDS.  8192 x 4096 x 4096 bf16, forward
// / dx / dW, bare products of uniform numbers: 258 / 275 / 276 us, 1.07 / 1.0 /
// 1.0 PFLOP/s.  Matrix instructions need less than half of the time, LDS reads
// and writes as much, and the barrier of each step keeps part of them apart.
// With several parts of the reduction (`splits`) each leaves its fp32 sums for
// join_parts_kernel.
template <typename E, bool kAcrossP, bool kAcrossQ, int kI, int kJ, int kWi,
          int kWj, bool kTiny>
__global__ void __launch_bounds__(kWi* kWj * 64)
    product_kernel(AtomoProduct a) {
  constexpr int kThreads = kWi * kWj * 64;
  constexpr int kFi = kI / kWi / 32, kFj = kJ / kWj / 32;
  __shared__ u32x4 lds[2][(kI + kJ) * kRowChunks];
  static_assert(kWi * kWj * pass_floats<kFi>() * 4 <= (int)sizeof(lds), "LDS");
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  const Work<E, kAcrossP, kAcrossQ, kI, kJ> work(a);

  f32x16 acc[kFi][kFj] = {};
  Stage<E, kI, kThreads, kAcrossP> sp;
  Stage<E, kJ, kThreads, kAcrossQ> sq;
  work.template load<kTiny>(a, 0, sp, sq);
  sp.store(lds[0]);
  sq.store(lds[0] + kI * kRowChunks);
  if (work.steps > 1) work.template load<kTiny>(a, 1, sp, sq);
  __syncthreads();
  const int wi = wave % kWi * (kI / kWi), wj = wave / kWi * (kJ / kWj);
  for (int s = 0; s < work.steps; ++s) {
    const u32x4* tp = lds[s & 1];
    const u32x4* tq = tp + kI * kRowChunks;
#pragma unroll
    for (int c = 0; c < kRowChunks; c += 2) {
      u32x4 fp[kFi], fq[kFj];
#pragma unroll
      for (int t = 0; t < kFi; ++t)
        fp[t] = tp[slot(wi + t * 32 + lane % 32, c + lane / 32)];
#pragma unroll
      for (int t = 0; t < kFj; ++t)
        fq[t] = tq[slot(wj + t * 32 + lane % 32, c + lane / 32)];
      multiply<E>(fp, fq, acc);
    }
    // the next step's tile, loaded a step ago, while the matrix instructions
    // drain (8192 x 4096 x 4096 bf16: 326 / 343 / 312 -> 314 / 301 / 296 us),
    // and the loads of the one after it
    if (s + 1 < work.steps) {
      u32x4* to = lds[(s + 1) & 1];
      sp.store(to);
      sq.store(to + kI * kRowChunks);
    }
    if (s + 2 < work.steps) work.template load<kTiny>(a, s + 2, sp, sq);
    __syncthreads();
  }
  write_tile<E>(a, work.part, work.i0 + wi, work.j0 + wj, acc,
                (float*)lds + wave * pass_floats<kFi>());
}

// Where 16-bit operands are aligned to 16 bytes and hold whole steps
// (direct_fits), memory is loaded straight into LDS, without registers in
// between, and an operand that lies across stays so there: the LDS reads
// transpose, 4 x 16 elements for each 16 lanes.  Nothing of a step is left to a
// wave but the loads' issue, a step ahead, and the fragments' reads.  The same
// sums in the same order as by registers.
typedef __attribute__((address_space(3))) void lds_void;

template <int kRows, int kThreads, bool kAcross>
struct Direct {
  static constexpr int kVecs = kRows * kRowChunks / kThreads;
  // Rows across: a k's row has kRows / 32 pieces of 64 bytes.  Sixteen lanes
  // read 32 bytes of four k each: neighbouring k have their pieces exchanged so
  // that these fall on all banks.
  __device__ static int turn(int k) {
    return kRows == 64 ? k >> 1 & 1 : k & 3;
  }
  __amdgpu_buffer_rsrc_t from;
  int at[kVecs];  // bytes, of the thread's vectors in step 0
  int step;       // bytes from one step to the next

  __device__ __forceinline__ Direct(const uint16_t* p, int64_t ld, int rows) {
    // offsets are below 2^31 (direct_fits) and in the matrix: rows from `rows`
    // on are read in the place of the last ones, for results that nobody keeps
    from = __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, 0x7FFFFFFF, 0x00027000);
    step = kAcross ? kRowBytes / 2 * (int)ld * 2 : kRowBytes;
#pragma unroll
    for (int s = 0; s < kVecs; ++s) {
      const int id = threadIdx.x + s * kThreads;
      if constexpr (!kAcross) {
        const int row = id / kRowChunks;
        const int c = (id % kRowChunks) ^ ((row ^ (row >> 3)) & 7);  // slot()
        at[s] = (min(row, rows - 1) * (int)ld + c * 8) * 2;
      } else {
        const int k = id / (kRows / 8), c = id % (kRows / 8);
        const int row = ((c / 4 ^ turn(k)) * 4 + c % 4) * 8;
        at[s] = (k * (int)ld + min(row, rows - 8)) * 2;
      }
    }
  }

  // a wave's 64 vectors lie one behind the other in LDS
  __device__ __forceinline__ void load(u32x4* tile, int s) const {
    u32x4* to = tile + threadIdx.x / 64 * 64;
#pragma unroll
    for (int v = 0; v < kVecs; ++v)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          from, (lds_void*)(to + v * kThreads), 16, at[v], s * step, 0, 0);
  }

  // of rows row..row + 31 the eight k of chunk c + lane / 32
  __device__ static __forceinline__ u32x4 fragment(const u32x4* tile, int row,
                                                   int c) {
    const int lane = threadIdx.x % 64;
    if constexpr (!kAcross) {
      return tile[slot(row + lane % 32, c + lane / 32)];
    } else {
      typedef short s16x4 __attribute__((ext_vector_type(4)));
      typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
      u32x4 out;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int k = (c + lane / 32) * 8 + h * 4 + lane % 16 / 4;
        const char* at = (const char*)tile + k * kRows * 2 +
                         (row / 32 ^ turn(k)) * 64 + lane % 32 / 16 * 32 +
                         lane % 4 * 8;
        const u32x2 r = __builtin_bit_cast(
            u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)at));
        out[2 * h] = r[0];
        out[2 * h + 1] = r[1];
      }
      return out;
    }
  }
};

// 8192 x 4096 x 4096 bf16, forward / dx / dW, bare products of uniform numbers:
// 221 / 234 / 223 us, where by registers they take 258 / 275 / 276.  Of normal
// numbers, in turn with a library's products: 225 / 248 / 241, the library's 180 /
// 206 / 242.  (The card's clock gives way to what the numbers cost: of zeros 182 /
// 213 / 203.)  In a pass of forward and backward with gelu and residual, passes
// in a row: 293 with epilogue and slope / 264 / 261, 0.94 / 1.04 / 1.05 PFLOP/s.
// Matrix instructions need half of that; LDS takes as long for its reads and
// writes, and the one barrier of a step keeps parts of the two apart: this
// arrangement's bound, not the card's, as the library's forward product shows.
// Half of the waves a phase behind the others, so that they read while those
// multiply: 222 / 269 / 260 of uniform numbers.  Two buffers of their own, so
// that the compiler sees that reads of one need not wait for loads into the other.
template <typename E, bool kAcrossP, bool kAcrossQ, int kI, int kJ, int kWi,
          int kWj>
__global__ void __launch_bounds__(kWi* kWj * 64)
    product_direct_kernel(AtomoProduct a) {
#if defined(__HIP_DEVICE_COMPILE__)  // LDS pointers are not the host's
  constexpr int kThreads = kWi * kWj * 64;
  constexpr int kFi = kI / kWi / 32, kFj = kJ / kWj / 32;
  __shared__ u32x4 even[(kI + kJ) * kRowChunks];
  __shared__ u32x4 odd[(kI + kJ) * kRowChunks];
  static_assert(kWi * kWj / 2 * pass_floats<kFi>() * 4 <= (int)sizeof(even), "LDS");
  const int wave = threadIdx.x / 64;
  const Work<E, kAcrossP, kAcrossQ, kI, kJ> work(a);
  using P = Direct<kI, kThreads, kAcrossP>;
  using Q = Direct<kJ, kThreads, kAcrossQ>;
  const P dp(work.p, a.ldp, work.rows_i);
  const Q dq(work.q, a.ldq, work.rows_j);
  const int wi = wave % kWi * (kI / kWi), wj = wave / kWi * (kJ / kWj);
  f32x16 acc[kFi][kFj] = {};
  const auto load = [&](u32x4* tile, int s) __attribute__((always_inline)) {
    s += work.begin;
    s = s < work.steps ? s : s - work.steps;
    dp.load(tile, s);
    dq.load(tile + kI * kRowChunks, s);
    __builtin_amdgcn_sched_barrier(0);  // before the step, not after it
  };
  const auto use = [&](const u32x4* tile) __attribute__((always_inline)) {
#pragma unroll
    for (int c = 0; c < kRowChunks; c += 2) {
      u32x4 fp[kFi], fq[kFj];
#pragma unroll
      for (int t = 0; t < kFi; ++t) fp[t] = P::fragment(tile, wi + t * 32, c);
#pragma unroll
      for (int t = 0; t < kFj; ++t)
        fq[t] = Q::fragment(tile + kI * kRowChunks, wj + t * 32, c);
      multiply<E>(fp, fq, acc);
    }
    // the wave's loads into the other buffer have arrived, then everybody's
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
    __syncthreads();
  };
  load(even, 0);
  __builtin_amdgcn_s_waitcnt(0x0F70);
  __syncthreads();
  int s = 0;
  for (; s + 1 < work.steps; s += 2) {
    load(odd, s + 1);
    use(even);
    if (s + 2 < work.steps) load(even, s + 2);
    use(odd);
  }
  if (s < work.steps) use(even);
  write_tile<E>(a, work.part, work.i0 + wi, work.j0 + wj, acc,
                (float*)(wave % 2 ? odd : even) + wave / 2 * pass_floats<kFi>());
#endif
}

// The same for fp32 operands on the bf16 matrix instructions, 16 times as fast
// as the fp32 ones: with x = a + b + c and y = a' + b' + c' (put_thirds) the
// six products aa', ab', ba', bb', ac', ca' are xy but for 2^-25 of it, less
// than fp32 loses by its sums, as long as the parts are normal numbers: what
// of an operand lies below 2^-126 may count as 0 (operands from 2^-101 on lose
// nothing).  2.7 times less time in matrix instructions: 8192 x 4096 x 4096
// forward in 1.4 ms, 0.2 PFLOP/s, above the 0.157 of the fp32 ones; 128 x 9216 x
// 4096, forward / dx / dW, with the parts joined, in 63 / 76 / 78 us (by fp32
// instructions 100 / 109 / 139).  There the weight's 151 MB take 27 us and the
// six products 39 at 1.5 PFLOP/s; splitting and LDS take as long, and the
// barriers keep them apart.  One buffer in LDS, so that three workgroups share a
// CU and fill each other's waits.
//
// Where a sum comes out infinite or NaN (0 times a split infinity is NaN, and
// so is what rounds up to one) the tile is made again, by fp32 instructions.
template <bool kAcrossP, bool kAcrossQ, int kI, int kJ, int kWi, int kWj>
__global__ void __launch_bounds__(kWi* kWj * 64)
    __attribute__((amdgpu_waves_per_eu(3))) product_thirds_kernel(AtomoProduct a) {
  constexpr int kThreads = kWi * kWj * 64;
  constexpr int kFi = kI / kWi / 32, kFj = kJ / kWj / 32;
  constexpr int kPlane = (kI + kJ) * kThirdBytes;
  __shared__ u32x4 lds[3 * kPlane / 16];
  static_assert(kWi * kWj * pass_floats<kFi>() * 4 <= (int)sizeof(lds), "LDS");
  char* tile_p = (char*)lds;
  char* tile_q = tile_p + kI * kThirdBytes;
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  const Work<F32, kAcrossP, kAcrossQ, kI, kJ> work(a);

  f32x16 acc[kFi][kFj] = {};
  Stage<F32, kI, kThreads, kAcrossP> sp;
  Stage<F32, kJ, kThreads, kAcrossQ> sq;
  work.template load<false>(a, 0, sp, sq);
  const int wi = wave % kWi * (kI / kWi), wj = wave / kWi * (kJ / kWj);
  for (int s = 0; s < work.steps; ++s) {
    sp.store_thirds(tile_p, kPlane);
    sq.store_thirds(tile_q, kPlane);
    __syncthreads();
    if (s + 1 < work.steps) work.template load<false>(a, s + 1, sp, sq);
#pragma unroll
    for (int c = 0; c < 4; c += 2) {
      u32x4 fp[3][kFi], fq[3][kFj];
#pragma unroll
      for (int h = 0; h < 3; ++h) {
#pragma unroll
        for (int t = 0; t < kFi; ++t)
          fp[h][t] = *(const u32x4*)(tile_p + h * kPlane +
                                     third_slot(wi + t * 32 + lane % 32,
                                                c + lane / 32) * 16);
#pragma unroll
        for (int t = 0; t < kFj; ++t)
          fq[h][t] = *(const u32x4*)(tile_q + h * kPlane +
                                     third_slot(wj + t * 32 + lane % 32,
                                                c + lane / 32) * 16);
      }
      // the small ones first
      multiply<BF16>(fp[2], fq[0], acc);
      multiply<BF16>(fp[0], fq[2], acc);
      multiply<BF16>(fp[1], fq[1], acc);
      multiply<BF16>(fp[1], fq[0], acc);
      multiply<BF16>(fp[0], fq[1], acc);
      multiply<BF16>(fp[0], fq[0], acc);
    }
    __syncthreads();
  }
  float odd = 0.f;  // NaN where a sum is not finite
#pragma unroll
  for (int ti = 0; ti < kFi; ++ti)
#pragma unroll
    for (int tj = 0; tj < kFj; ++tj)
#pragma unroll
      for (int e = 0; e < 16; ++e) odd += acc[ti][tj][e] * 0.f;
  if (__ballot(odd != odd) != 0) {
    // 32 x 32 after 32 x 32: rare, so short rather than fast
#pragma unroll
    for (int ti = 0; ti < kFi; ++ti)
#pragma unroll
      for (int tj = 0; tj < kFj; ++tj) {
        const int64_t i = min(wi + ti * 32 + lane % 32, work.rows_i - 1);
        const int64_t j = min(wj + tj * 32 + lane % 32, work.rows_j - 1);
        const uint32_t* x = work.p + (kAcrossP ? i : i * a.ldp);
        const uint32_t* y = work.q + (kAcrossQ ? j : j * a.ldq);
        acc[ti][tj] = f32x16{};
        // lane halves take neighbouring k
        for (int k = 0; k < work.ks; k += 2) {
          const int64_t at = min(k + lane / 32, work.ks - 1);
          float u = __uint_as_float(x[kAcrossP ? at * a.ldp : at]);
          float v = __uint_as_float(y[kAcrossQ ? at * a.ldq : at]);
          u = k + lane / 32 < work.ks ? u : 0.f;
          v = k + lane / 32 < work.ks ? v : 0.f;
          acc[ti][tj] = __builtin_amdgcn_mfma_f32_32x32x2f32(u, v, acc[ti][tj],
                                                             0, 0, 0);
        }
      }
  }
  write_tile<F32>(a, work.part, work.i0 + wi, work.j0 + wj, acc,
                  (float*)lds + wave * pass_floats<kFi>());
}

constexpr int kThreads = 256;

// The parts' sums, added in order, and the epilogue; a thread four neighbours.
// Bound by the memory: 16 parts of 128 x 4096 in 7.5 us.
template <typename E>
__global__ void __launch_bounds__(kThreads) join_parts_kernel(AtomoProduct a) {
  const int64_t fours = a.ld_part / 4;
  const int64_t id = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  const int64_t j = id / fours;
  const int i = (int)(id % fours) * 4;
  if (j >= a.nj) return;
  const Four<typename E::Raw> bias = bias_of<E>(a, i);
  const Four<typename E::Raw> residual = residual_of<E>(a, j, i);
  float sum[4] = {};
#pragma unroll 4
  for (int part = 0; part < a.splits; ++part) {
    const float4 v = *(const float4*)(a.partial +
                                      ((int64_t)part * a.nj + j) * a.ld_part + i);
    sum[0] += v.x;
    sum[1] += v.y;
    sum[2] += v.z;
    sum[3] += v.w;
  }
  finish<E>(a, j, i, sum, bias, residual);
}

// Few rows, bound by the memory (1 x 9216 -> 4096 bf16 in 13 us, 5.8 TB/s; in
// tiles 16 us; fp32 in 22 us, 6.8 TB/s, part of it from the cache): the weight
// is read once, by waves that each take kN of its rows and all of x's kM; a lane
// takes every 64th 16 bytes.
template <typename E, int kM, int kN>
__global__ void __launch_bounds__(kThreads) few_rows_kernel(AtomoProduct a) {
  using Raw = typename E::Raw;
  constexpr int kC = E::kChunk;
  const int lane = threadIdx.x % 64;
  const int n0 = (blockIdx.x * (kThreads / 64) + (int)(threadIdx.x / 64)) * kN;
  if (n0 >= a.ni) return;
  const Raw* w[kN];
  const Raw* x[kM];
#pragma unroll
  for (int n = 0; n < kN; ++n)
    w[n] = (const Raw*)a.p + min(n0 + n, a.ni - 1) * a.ldp;
#pragma unroll
  for (int m = 0; m < kM; ++m)
    x[m] = (const Raw*)a.q + min(m, a.nj - 1) * a.ldq;
  float sum[kN][kM] = {};
  const auto value = [](const u32x4& v, int e) {
    if constexpr (kC == 4)
      return E::widen(v[e]);
    else
      return E::widen((uint16_t)(v[e / 2] >> (e % 2 * 16)));
  };
  const auto load = [](const Raw* at) -> u32x4 {
    if constexpr (kC == 4)
      return *(const u32x4_a4*)at;
    else
      return *(const u32x4_a2*)at;
  };
  const int whole = a.nk / kC * kC;
  constexpr int kUnroll = kM <= 2 ? 4 : 2;
  int k = lane * kC;
  for (; k + (kUnroll - 1) * 64 * kC < whole; k += kUnroll * 64 * kC) {
    u32x4 vw[kUnroll][kN];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
#pragma unroll
      for (int n = 0; n < kN; ++n) vw[u][n] = load(w[n] + k + u * 64 * kC);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
#pragma unroll
      for (int m = 0; m < kM; ++m) {
        const u32x4 vx = load(x[m] + k + u * 64 * kC);
#pragma unroll
        for (int e = 0; e < kC; ++e)
#pragma unroll
          for (int n = 0; n < kN; ++n)
            sum[n][m] += value(vw[u][n], e) * value(vx, e);
      }
  }
  for (; k < whole; k += 64 * kC)
#pragma unroll
    for (int n = 0; n < kN; ++n) {
      const u32x4 vw = load(w[n] + k);
#pragma unroll
      for (int m = 0; m < kM; ++m) {
        const u32x4 vx = load(x[m] + k);
#pragma unroll
        for (int e = 0; e < kC; ++e) sum[n][m] += value(vw, e) * value(vx, e);
      }
    }
  if (whole + lane < a.nk) {
#pragma unroll
    for (int n = 0; n < kN; ++n)
#pragma unroll
      for (int m = 0; m < kM; ++m)
        sum[n][m] += E::widen(w[n][whole + lane]) * E::widen(x[m][whole + lane]);
  }
#pragma unroll
  for (int n = 0; n < kN; ++n)
#pragma unroll
    for (int m = 0; m < kM; ++m) {
#pragma unroll
      for (int off = 32; off > 0; off >>= 1)
        sum[n][m] += __shfl_xor(sum[n][m], off, 64);
    }
  // lane m writes row m
#pragma unroll
  for (int m = 0; m < kM; ++m) {
    if (lane != m || m >= a.nj) continue;
#pragma unroll
    for (int n = 0; n < kN; ++n) {
      if (n0 + n >= a.ni) break;
      float h = sum[n][m], d;
      if (a.bias) h += E::widen(((const Raw*)a.bias)[n0 + n]);
      h = activate<E::kChunk == 8>(a.act, h, &d);
      if (a.slope) ((float*)a.slope)[(int64_t)m * a.ni + n0 + n] = d;
      if (a.residual)
        h += E::widen(((const Raw*)a.residual)[m * a.ldr + n0 + n]);
      ((Raw*)a.out)[m * a.ldo + n0 + n] = output<E>(a, h);
    }
  }
}

// dp, and the sums of the columns of a block of rows.  64 lanes take 64 times
// kV neighbours of a row, the waves every kDpWaves-th row.  Bound by the
// memory: 8192 x 4096 bf16 with slopes in 63 us, 4.3 TB/s.  kV is four, or one
// where four would leave most CUs without a workgroup: 128 x 4096 fp32 in 6.5 us
// (by fours 13), 128 x 800 in 5 (9).
//
// dp is rounded to the operands' type, as the products' operand; db is summed
// before.  Where the slope is 0 or 1 nothing is rounded.  Else, of 8192 x 4096 x
// 4096 bf16 with gelu, dx and dW are 0.0023 of their norm off 64 bits: 0.0017 by
// the rounding of the results, as much by that of dp.  To keep dp's lower part
// as an operand of its own would double both products, 0.5 of 0.86 ms more.
constexpr int kDpWaves = 16;

template <typename E, int kV>
__global__ void __launch_bounds__(kDpWaves * 64)
    linear_dp_kernel(AtomoLinearDp a) {
  using Raw = typename E::Raw;
  __shared__ float lds[kDpWaves][64 * kV];
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  const int c = (blockIdx.x * 64 + lane) * kV;
  const int n = min(kV, a.columns - c);
  const int first = blockIdx.y * a.block_rows;
  const int last = min(a.rows, first + a.block_rows);
  const Raw* dy = (const Raw*)a.dy;
  const bool by_output = a.slope && a.by_output;
  const bool by_slope = a.slope && !a.by_output;
  float sum[kV] = {};
  // four rows are read before the first is used
  constexpr int kDepth = 4;
  for (int r0 = first + wave; r0 < last; r0 += kDpWaves * kDepth) {
    if (n <= 0) break;
    Some<Raw, kV> v[kDepth], y[kDepth];
    Some<float, kV> s[kDepth];
    const auto load = [&](int n) {
#pragma unroll
      for (int u = 0; u < kDepth; ++u) {
        const int64_t r = min(r0 + u * kDpWaves, last - 1);
        const int64_t at = r * a.columns + c;
        v[u] = load_some<kV>(dy + r * a.ld_dy + c, n);
        if (by_output) y[u] = load_some<kV>((const Raw*)a.slope + at, n);
        if (by_slope) s[u] = load_some<kV>((const float*)a.slope + at, n);
      }
    };
    // apart, so that whole ones are read without a branch in between
    if (n == kV)
      load(kV);
    else
      load(n);
#pragma unroll
    for (int u = 0; u < kDepth; ++u) {
      const int r = r0 + u * kDpWaves;
      if (r >= last) break;
#pragma unroll
      for (int e = 0; e < kV; ++e) {
        float d = E::widen(v[u].v[e]);
        if (by_output)
          d = relu_is_off<E>(y[u].v[e]) ? 0.f : d;
        else if (by_slope)
          d *= s[u].v[e];
        v[u].v[e] = E::narrow(d);
        sum[e] += d;
      }
      if (a.dp)
        store_some<kV>((Raw*)a.dp + (int64_t)r * a.columns + c, n, v[u]);
    }
  }
  if (!a.db) return;
#pragma unroll
  for (int e = 0; e < kV; ++e) lds[wave][lane * kV + e] = sum[e];
  __syncthreads();
  if (threadIdx.x < 64 * kV) {
    float all = 0.f;
#pragma unroll
    for (int w = 0; w < kDpWaves; ++w) all += lds[w][threadIdx.x];
    const int column = blockIdx.x * 64 * kV + threadIdx.x;
    if (column < a.columns) {
      if (a.row_blocks == 1)
        ((Raw*)a.db)[column] = E::narrow(all);
      else
        a.partial[(int64_t)blockIdx.y * a.columns + column] = all;
    }
  }
}

// the blocks' column sums, 64 columns by 16 waves
template <typename E>
__global__ void __launch_bounds__(kDpWaves * 64)
    linear_db_kernel(const float* __restrict__ partial, int blocks, int columns,
                     typename E::Raw* __restrict__ db) {
  __shared__ float lds[kDpWaves][64];
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  const int c = blockIdx.x * 64 + lane;
  float sum = 0.f;
  if (c < columns)
    for (int b = wave; b < blocks; b += kDpWaves)
      sum += partial[(int64_t)b * columns + c];
  lds[wave][lane] = sum;
  __syncthreads();
  if (wave == 0 && c < columns) {
    float all = 0.f;
#pragma unroll
    for (int w = 0; w < kDpWaves; ++w) all += lds[w][lane];
    db[c] = E::narrow(all);
  }
}

template <typename E, bool kAcrossP, bool kAcrossQ, int kI, int kJ, int kWi,
          int kWj, bool kTiny>
void launch_product(const AtomoProduct& a, hipStream_t stream) {
  const int64_t tiles = (int64_t)((a.ni + kI - 1) / kI) * ((a.nj + kJ - 1) / kJ);
  const dim3 grid((unsigned)(tiles * a.splits)), block(kWi * kWj * 64);
  if constexpr (E::kChunk == 4 && !kTiny)
    hipLaunchKernelGGL((product_thirds_kernel<kAcrossP, kAcrossQ, kI, kJ, kWi, kWj>),
                       grid, block, 0, stream, a);
  else if (!kTiny && a.direct) {
    if constexpr (E::kChunk == 8 && !kTiny)
      hipLaunchKernelGGL(
          (product_direct_kernel<E, kAcrossP, kAcrossQ, kI, kJ, kWj, kWi>), grid,
          block, 0, stream, a);
  } else {
    hipLaunchKernelGGL((product_kernel<E, kAcrossP, kAcrossQ, kI, kJ, kWi, kWj, kTiny>),
                       grid, block, 0, stream, a);
  }
}

template <typename E, int kI, int kJ, int kWi, int kWj, bool kTiny = false>
void product(const AtomoProduct& a, hipStream_t stream) {
  if (a.form == ATOMO_FORWARD)
    launch_product<E, false, false, kI, kJ, kWi, kWj, kTiny>(a, stream);
  else if (a.form == ATOMO_GRAD_X)
    launch_product<E, true, false, kI, kJ, kWi, kWj, kTiny>(a, stream);
  else
    launch_product<E, true, true, kI, kJ, kWi, kWj, kTiny>(a, stream);
}

template <typename E, int kM>
void few_rows(const AtomoProduct& a, hipStream_t stream) {
  constexpr int kN = 2;
  const int per = kThreads / 64 * kN;
  hipLaunchKernelGGL((few_rows_kernel<E, kM, kN>), dim3((a.ni + per - 1) / per),
                     dim3(kThreads), 0, stream, a);
}

template <typename E>
void product(const AtomoProduct& a, hipStream_t stream) {
  if (a.plan == ATOMO_PLAN_FEW_ROWS) {
    if (a.nj <= 1)
      few_rows<E, 1>(a, stream);
    else if (a.nj <= 2)
      few_rows<E, 2>(a, stream);
    else if constexpr (E::kChunk == 4)
      few_rows<E, 4>(a, stream);
    return;
  }
  if (a.plan == ATOMO_PLAN_TINY)
    product<E, 64, 64, 2, 2, true>(a, stream);
  else if (a.plan == ATOMO_PLAN_64)
    product<E, 64, 64, 2, 2>(a, stream);
  else if (a.plan == ATOMO_PLAN_128)
    product<E, 128, 128, 2, 2>(a, stream);
  else if constexpr (E::kChunk == 8)
    product<E, 256, 256, 2, 4>(a, stream);
  if (a.splits > 1) {
    const int64_t fours = a.ld_part / 4 * a.nj;
    hipLaunchKernelGGL((join_parts_kernel<E>),
                       dim3((unsigned)((fours + kThreads - 1) / kThreads)),
                       dim3(kThreads), 0, stream, a);
  }
}

template <typename E, int kV>
void launch_dp(const AtomoLinearDp& a, hipStream_t stream) {
  const int wide = 64 * kV;
  hipLaunchKernelGGL((linear_dp_kernel<E, kV>),
                     dim3((a.columns + wide - 1) / wide, a.row_blocks),
                     dim3(kDpWaves * 64), 0, stream, a);
}

template <typename E>
void linear_dp(const AtomoLinearDp& a, hipStream_t stream) {
  if ((int64_t)(a.columns + 255) / 256 * a.row_blocks < 128)
    launch_dp<E, 1>(a, stream);
  else
    launch_dp<E, 4>(a, stream);
  if (a.db && a.row_blocks > 1)
    hipLaunchKernelGGL((linear_db_kernel<E>), dim3((a.columns + 63) / 64),
                       dim3(kDpWaves * 64), 0, stream, a.partial, a.row_blocks,
                       a.columns, (typename E::Raw*)a.db);
}

// What a step of 128 bytes of the reduction costs a workgroup, in us: alone on
// its CU, where it waits for its loads, and as its share of a full one; by
// kernel (fp32, 16 bits by registers, straight into LDS), form and tile (64, 128,
// 256).  Measured on bare products of uniform numbers, 16 to 8192 by 10 to 4096
// by 500 to 9216; the choices that follow from it, and what lies next to them:
//   1024 x 1024 x 1024 bf16 forward: 64, one part 8 us; 128, two parts 16
//   2048 x 2048 x 2048 bf16 forward: 128, one part 30 us; two parts 38
//   8192 x 4096 x 4096 bf16 forward: 256, one part 221 us; 128 267; 64 421
//   512 x 512 x 4096 bf16 forward: 64, eight parts 13 us; four 12, two 15
//   128 x 9216 -> 4096 fp32 forward: 128, 16 parts 63 us; 8 or 32 parts 75
struct Step {
  float alone, shared;
};
constexpr Step kStep[3][3][3] = {
    {{{0.90f, 0.56f}, {1.95f, 1.50f}, {}},
     {{1.15f, 0.57f}, {1.85f, 1.50f}, {}},
     {{1.40f, 0.83f}, {1.90f, 1.60f}, {}}},
    {{{0.55f, 0.29f}, {0.90f, 0.98f}, {2.40f, 2.40f}},
     {{0.75f, 0.34f}, {0.95f, 1.05f}, {2.35f, 2.35f}},
     {{0.95f, 0.60f}, {1.00f, 1.10f}, {2.30f, 2.30f}}},
    {{{0.37f, 0.25f}, {0.90f, 0.52f}, {1.50f, 1.75f}},
     {{0.37f, 0.25f}, {1.10f, 0.56f}, {1.80f, 1.88f}},
     {{0.37f, 0.25f}, {1.05f, 0.55f}, {1.70f, 1.79f}}}};
constexpr float kTileEnd[3] = {0.25f, 1.4f, 6.f};  // a tile's epilogue

float cost_of(const AtomoProduct& a, int tile, int64_t splits, int steps) {
  constexpr int kCus = 256;
  const int size = 64 << tile;
  const int64_t tiles =
      (int64_t)((a.ni + size - 1) / size) * ((a.nj + size - 1) / size);
  const Step& step =
      kStep[a.type == ATOMO_F32 ? 0 : a.direct ? 2 : 1][a.form][tile];
  const float per_cu = (float)((tiles * splits + kCus - 1) / kCus);
  float each = step.shared * per_cu;
  if (each < step.alone) each = step.alone;
  float us = each * (float)((steps + splits - 1) / splits) +
             kTileEnd[tile] * per_cu;
  // a launch more, and the sums written and read again at 5.5 TB/s
  if (splits > 1) us += 3.5f + (float)a.ni * a.nj * splits * (8 / 5.5e6f);
  return us;
}

// Whether an operand may be loaded straight into LDS: 16-byte vectors at
// aligned places, eight rows or eight k at once, whole steps of 64 k, and byte
// offsets within a workgroup's part below 2^31.
bool direct_fits(const void* p, int64_t ld, int rows, int nk, bool across) {
  if ((uintptr_t)p % 16 != 0 || ld % 8 != 0 || nk % 64 != 0) return false;
  if (across) return rows % 8 == 0 && ld < ((int64_t)1 << 29) / nk;
  return ld < (int64_t)1 << 21 && nk < 1 << 29;
}

}  // namespace

#define ATOMO_BY_TYPE(call)                         \
  if (a->type == ATOMO_F32)                         \
    call<F32>(*a, stream);                          \
  else if (a->type == ATOMO_BF16)                   \
    call<BF16>(*a, stream);                         \
  else                                              \
    call<F16>(*a, stream);

extern "C" {

void atomo_product_plan(AtomoProduct* a) {
  a->direct = 0;
  a->splits = 1;
  a->k_part = a->nk;
  a->ld_part = (a->ni + 3) / 4 * 4;
  a->bare = a->act == ATOMO_ACT_NONE && !a->bias && !a->residual && !a->slope;
  // Beyond, its vector instructions bound it, where tiles grow little with the
  // rows.  At the border, 2 rows so / 3 in tiles, bf16: 512 -> 512 2.9 / 4.3 us,
  // 2048 -> 2048 4.5 / 6.3, 4096 -> 4096 8.3 / 9.8, 9216 -> 4096 20 / 16; 4 rows
  // so / 5 in tiles, fp32: 4.5 / 7.4, 12 / 11, 25 / 23, 49 / 45.
  if (a->form == ATOMO_FORWARD && a->nj <= (a->type == ATOMO_F32 ? 4 : 2)) {
    a->plan = ATOMO_PLAN_FEW_ROWS;
    return;
  }
  // a vector of the reduction, or four rows that lie across, are read at once
  if ((a->form != ATOMO_GRAD_W && a->nk < 8) ||
      (a->form != ATOMO_FORWARD && a->ni < 4) ||
      (a->form == ATOMO_GRAD_W && a->nj < 4)) {
    a->plan = ATOMO_PLAN_TINY;
    return;
  }
  a->direct = a->type != ATOMO_F32 &&
              direct_fits(a->p, a->ldp, a->ni, a->nk, a->form != ATOMO_FORWARD) &&
              direct_fits(a->q, a->ldq, a->nj, a->nk, a->form == ATOMO_GRAD_W);
  const int step = kRowBytes / (a->type == ATOMO_F32 ? 4 : 2);
  const int steps = (a->nk + step - 1) / step;
  float least = 0.f;
  int64_t splits = 0;
  for (int tile = 0; tile < (a->type == ATOMO_F32 ? 2 : 3); ++tile)
    for (const int n : {1, 2, 3, 4, 5, 6, 7, 8, 10, 12, 14, 16, 20, 24, 32}) {
      if (n > 1 && n * 4 > steps) break;  // parts of four steps at least
      const float us = cost_of(*a, tile, n, steps);
      if (splits && us >= least) continue;
      least = us;
      splits = n;
      a->plan = ATOMO_PLAN_64 + tile;
    }
  if (splits > 1) {
    const int part = (int)((steps + splits - 1) / splits);
    a->k_part = part * step;
    a->splits = (steps + part - 1) / part;
    a->bare = 1;
  }
}

void atomo_product_launch(const AtomoProduct* a, hipStream_t stream) {
  ATOMO_BY_TYPE(product)
}

void atomo_linear_dp_launch(const AtomoLinearDp* a, hipStream_t stream) {
  ATOMO_BY_TYPE(linear_dp)
}

}  // extern "C"
