// Kernels on the logits of a classifier for MI355X (gfx950): log probability
// of given classes with entropy and top alternatives, and distillation from
// a teacher's top logits with its gradient.
//
// Mathematics, for a row z of V logits (m = max z, d = z - m <= 0):
//   S   = sum exp(d)            log softmax(z)_v = d_v - log S
//   T   = sum d exp(d)          entropy          = log S - T / S
//   S_t = sum exp(d / tau)      softmax(z / tau) = exp(d / tau) / S_t
// and for a teacher's K values t at classes i, q = softmax(t / tau) over the
// K, entries of one class added up:
//   KD  = tau^2 sum_c q_c (log q_c - log softmax(z / tau)_c)
//   row = w KD + (1 - w) (log S - d_y)
//   dz  = w tau (softmax(z / tau) - q) + (1 - w) (softmax(z) - onehot_y)
//
// Everything is held in 32-bit floats; 16-bit logits are widened as they are
// read and the gradient is rounded once, as it is written.
//
// Rows without a finite maximum: a row of -inf only has no distribution; its
// log probabilities are -inf, its entropy 0, its loss and gradient 0.  A row
// with NaN or +inf gives NaN.

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include <cstdint>

#include "logit_kernels.h"

#define WAVE 64

namespace {

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kInf = __builtin_huge_valf();
constexpr int kThreads = 256;
constexpr int kWaves = kThreads / WAVE;
constexpr int kTopMax = ATOMO_LOGIT_TOP_MAX;

__device__ __forceinline__ float widen(float x) { return x; }
__device__ __forceinline__ float widen(__half x) { return __half2float(x); }
__device__ __forceinline__ float widen(__hip_bfloat16 x) {
  return __bfloat162float(x);
}
template <typename T>
__device__ __forceinline__ T narrow(float x);
template <>
__device__ __forceinline__ float narrow<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half narrow<__half>(float x) {
  return __float2half(x);
}
template <>
__device__ __forceinline__ __hip_bfloat16 narrow<__hip_bfloat16>(float x) {
  return __float2bfloat16(x);
}

// e^d for d <= 0 (or NaN); e^-inf = 0
__device__ __forceinline__ float exp_of(float d) {
  return __builtin_amdgcn_exp2f(d * kLog2e);
}

// Order of the classes by logit: whole numbers that rise with the value, NaN
// above all, -0 equal to +0; the lowest class first among equals.  No class
// has key 0.
__device__ __forceinline__ uint32_t order_of(float x) {
  if (x != x) return 0xFFFFFFFFu;
  const uint32_t b = __float_as_uint(x + 0.0f);
  return (b >> 31) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ uint64_t key_of(float x, uint32_t column) {
  return ((uint64_t)order_of(x) << 32) | (0xFFFFFFFFu - column);
}
__device__ __forceinline__ uint32_t column_of(uint64_t key) {
  return 0xFFFFFFFFu - (uint32_t)key;
}

// Maximum and the sums relative to it; joined pairwise in a fixed order.
struct Stat {
  float m, s, t;
};

// 0 stands in for a maximum of -inf: exp(-inf - 0) is 0, not NaN
__device__ __forceinline__ float origin(float m) { return m == -kInf ? 0.f : m; }

__device__ __forceinline__ Stat join(Stat a, Stat b) {
  Stat r;
  r.m = fmaxf(a.m, b.m);
  const float o = origin(r.m);
  // the floor keeps 0 * -inf out of t
  const float da = fmaxf(a.m - o, -1e30f), db = fmaxf(b.m - o, -1e30f);
  const float fa = exp_of(da), fb = exp_of(db);
  r.s = a.s * fa + b.s * fb;
  r.t = (a.t + da * a.s) * fa + (b.t + db * b.s) * fb;
  return r;
}

__device__ __forceinline__ Stat wave_join(Stat v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    Stat o;
    o.m = __shfl_xor(v.m, off, WAVE);
    o.s = __shfl_xor(v.s, off, WAVE);
    o.t = __shfl_xor(v.t, off, WAVE);
    // the same operand order in both lanes of a pair: one result for all
    v = (threadIdx.x & off) ? join(o, v) : join(v, o);
  }
  return v;
}

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v = fmaxf(v, __shfl_xor(v, off, WAVE));
  return v;
}
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, WAVE);
  return v;
}
__device__ __forceinline__ uint64_t wave_max_key(uint64_t v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    const uint64_t o = __shfl_xor((unsigned long long)v, off, WAVE);
    v = o > v ? o : v;
  }
  return v;
}

__device__ __forceinline__ float block_max(float v, float* lds) {
  v = wave_max(v);
  __syncthreads();
  if (threadIdx.x % WAVE == 0) lds[threadIdx.x / WAVE] = v;
  __syncthreads();
  float r = lds[0];
#pragma unroll
  for (int i = 1; i < kWaves; ++i) r = fmaxf(r, lds[i]);
  return r;
}
__device__ __forceinline__ float block_sum(float v, float* lds) {
  v = wave_sum(v);
  __syncthreads();
  if (threadIdx.x % WAVE == 0) lds[threadIdx.x / WAVE] = v;
  __syncthreads();
  float r = lds[0];
#pragma unroll
  for (int i = 1; i < kWaves; ++i) r += lds[i];
  return r;
}

// log softmax of one logit; `o` = origin(m)
__device__ __forceinline__ float log_prob(float z, float m, float log_s) {
  if (m == -kInf && log_s == -kInf) return -kInf;  // an empty row
  return (z - origin(m)) - log_s;
}

// ---------------------------------------------------------------------------
// log probability, entropy, top alternatives: one workgroup a row
// ---------------------------------------------------------------------------
template <typename T>
__global__ void __launch_bounds__(kThreads)
    label_logprobs_kernel(const T* __restrict__ logits, int64_t row_stride,
                          int64_t rows, int classes,
                          const int64_t* __restrict__ labels, int64_t ignore,
                          int top, float* __restrict__ logprob,
                          float* __restrict__ entropy,
                          float* __restrict__ top_logprob,
                          int64_t* __restrict__ top_index) {
  __shared__ float lds[kWaves];
  __shared__ uint64_t lds_key[kWaves];
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const T* z = logits + row * row_stride;
    float m = -kInf;
    for (int c = threadIdx.x; c < classes; c += kThreads)
      m = fmaxf(m, widen(z[c]));
    m = block_max(m, lds);
    const float o = origin(m);
    float s = 0.f, t = 0.f;
    for (int c = threadIdx.x; c < classes; c += kThreads) {
      const float d = widen(z[c]) - o;
      const float e = exp_of(d);
      s += e;
      t += e * fmaxf(d, -1e30f);
    }
    s = block_sum(s, lds);
    t = block_sum(t, lds);
    const float log_s = logf(s);
    if (threadIdx.x == 0) {
      entropy[row] = s == 0.f ? 0.f : log_s - t / s;
      if (labels != nullptr) {
        const int64_t y = labels[row];
        float lp = __builtin_nanf("");
        if (y == ignore)
          lp = 0.f;
        else if (y >= 0 && y < classes)
          lp = log_prob(widen(z[y]), m, log_s);
        logprob[row] = lp;
      }
    }
    uint64_t last = ~0ull;
    for (int k = 0; k < top; ++k) {
      uint64_t best = 0;
      for (int c = threadIdx.x; c < classes; c += kThreads) {
        const uint64_t key = key_of(widen(z[c]), c);
        if (key < last && key > best) best = key;
      }
      best = wave_max_key(best);
      __syncthreads();
      if (threadIdx.x % WAVE == 0) lds_key[threadIdx.x / WAVE] = best;
      __syncthreads();
      best = lds_key[0];
#pragma unroll
      for (int i = 1; i < kWaves; ++i) best = max(best, lds_key[i]);
      if (threadIdx.x == 0) {
        const uint32_t c = column_of(best);
        top_index[row * top + k] = c;
        top_logprob[row * top + k] = log_prob(widen(z[c]), m, log_s);
      }
      last = best;
    }
  }
}

// ---------------------------------------------------------------------------
// distillation
// ---------------------------------------------------------------------------

// A teacher's row.
struct Sparse {
  float value[kTopMax];  // t, then log q
  int column[kTopMax];   // -1: absent
  float share[kTopMax];
  float red[kWaves];
  int bad;
};

__global__ void __launch_bounds__(1024)
    count_rows_kernel(const int64_t* __restrict__ labels, int64_t rows,
                      int64_t ignore, float* __restrict__ inverse) {
  __shared__ int lds[1024 / WAVE];
  int n = 0;
  for (int64_t i = threadIdx.x; i < rows; i += 1024) n += labels[i] != ignore;
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) n += __shfl_xor(n, off, WAVE);
  if (threadIdx.x % WAVE == 0) lds[threadIdx.x / WAVE] = n;
  __syncthreads();
  if (threadIdx.x == 0) {
    int all = 0;
    for (int i = 0; i < 1024 / WAVE; ++i) all += lds[i];
    *inverse = 1.0f / (float)(all > 0 ? all : 1);
  }
}

__global__ void __launch_bounds__(1024)
    sum_rows_kernel(const float* __restrict__ row_loss, int64_t rows,
                    const float* __restrict__ inverse, float factor,
                    float* __restrict__ loss) {
  __shared__ float lds[1024 / WAVE];
  // scaled before they are added: a mean of huge rows stays finite
  const float each = inverse ? *inverse : factor;
  float v = 0.f;
  for (int64_t i = threadIdx.x; i < rows; i += 1024) v += row_loss[i] * each;
  v = wave_sum(v);
  if (threadIdx.x % WAVE == 0) lds[threadIdx.x / WAVE] = v;
  __syncthreads();
  if (threadIdx.x == 0) {
    float all = 0.f;
    for (int i = 0; i < 1024 / WAVE; ++i) all += lds[i];
    *loss = all;
  }
}

// Loads the teacher's row, leaves q in `share` and the class in `column`.
// Returns the sum of q: 1, or 0 where no entry has a finite value, or NaN.
__device__ float load_teacher(Sparse& sp, const float* values,
                              const int64_t* index, int k, int classes,
                              float inv_tau) {
  __syncthreads();
  if (threadIdx.x == 0) sp.bad = 0;
  float m = -kInf;
  for (int j = threadIdx.x; j < k; j += kThreads) {
    const float v = values[j];
    sp.value[j] = v;
    m = fmaxf(m, v);
  }
  m = block_max(m, sp.red);
  const float o = origin(m);
  float s = 0.f;
  for (int j = threadIdx.x; j < k; j += kThreads) {
    const float v = sp.value[j];
    s += exp_of((v - o) * inv_tau);
    int c = -1;
    if (v != -kInf) {
      const int64_t i = index[j];
      if (i >= 0 && i < classes)
        c = (int)i;
      else
        sp.bad = 1;
    }
    sp.column[j] = c;
  }
  s = block_sum(s, sp.red);  // its barriers also publish column and bad
  const float log_s = logf(s);
  for (int j = threadIdx.x; j < k; j += kThreads) {
    const float lq = sp.column[j] < 0 ? -kInf : (sp.value[j] - o) * inv_tau - log_s;
    sp.value[j] = lq;
    sp.share[j] = sp.column[j] < 0 ? 0.f : exp_of(lq);
  }
  __syncthreads();
  if (sp.bad) return __builtin_nanf("");
  return s == 0.f ? 0.f : (s == s ? 1.f : s);
}

// q of entry j's class, or -1 where an earlier entry stands for that class
__device__ __forceinline__ float merged_share(const Sparse& sp, int j, int k,
                                              bool* alone) {
  const int c = sp.column[j];
  if (c < 0) return -1.f;
  float q = 0.f;
  *alone = true;
  for (int i = 0; i < k; ++i) {
    if (sp.column[i] != c) continue;
    if (i < j) return -1.f;
    if (i > j) *alone = false;
    q += sp.share[i];
  }
  return q;
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
    distill_loss_kernel(const T* __restrict__ logits, int64_t row_stride,
                        int64_t rows, int classes,
                        const float* __restrict__ values,
                        const int64_t* __restrict__ index, int k,
                        const int64_t* __restrict__ labels, int64_t ignore,
                        float tau, float weight, float* __restrict__ row_loss,
                        float* __restrict__ stats) {
  __shared__ Sparse sp;
  __shared__ float lds[kWaves];
  const float inv_tau = 1.0f / tau;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const int64_t y = labels ? labels[row] : 0;
    if (labels && y == ignore) {
      if (threadIdx.x == 0) row_loss[row] = 0.f;
      continue;
    }
    const T* z = logits + row * row_stride;
    float m = -kInf;
    for (int c = threadIdx.x; c < classes; c += kThreads)
      m = fmaxf(m, widen(z[c]));
    m = block_max(m, lds);
    const float o = origin(m);
    float s1 = 0.f, st = 0.f;
    for (int c = threadIdx.x; c < classes; c += kThreads) {
      const float d = widen(z[c]) - o;
      s1 += exp_of(d);
      st += exp_of(d * inv_tau);
    }
    s1 = block_sum(s1, lds);
    st = block_sum(st, lds);
    const float q_sum =
        load_teacher(sp, values + row * k, index + row * k, k, classes, inv_tau);
    const float log_st = logf(st);
    float kd = 0.f;
    for (int j = threadIdx.x; j < k; j += kThreads) {
      bool alone;
      const float q = merged_share(sp, j, k, &alone);
      if (q > 0.f) {
        const float lp = (widen(z[sp.column[j]]) - o) * inv_tau - log_st;
        kd += q * ((alone ? sp.value[j] : logf(q)) - lp);
      } else if (q != q) {
        kd = q;
      }
    }
    kd = block_sum(kd, lds);
    if (threadIdx.x == 0) {
      float loss = 0.f;
      if (s1 != 0.f) {  // a row of -inf only has no loss
        if (weight != 0.f)
          loss = weight * tau * tau * (q_sum != q_sum ? q_sum : kd);
        if (labels && weight != 1.f) {
          if (y >= 0 && y < classes)
            loss += (1.f - weight) * (logf(s1) - (widen(z[y]) - o));
          else
            loss = __builtin_nanf("");
        }
      }
      row_loss[row] = loss;
      stats[row * 3] = m;
      stats[row * 3 + 1] = s1;
      stats[row * 3 + 2] = st;
    }
  }
}

// dz from the row's statistics.  `up` is the loss's gradient: one value, or
// one a row.
template <typename T>
__global__ void __launch_bounds__(kThreads)
    distill_grad_kernel(const T* __restrict__ logits, int64_t row_stride,
                        int64_t rows, int classes,
                        const float* __restrict__ values,
                        const int64_t* __restrict__ index, int k,
                        const int64_t* __restrict__ labels, int64_t ignore,
                        float tau, float weight,
                        const float* __restrict__ stats,
                        const float* __restrict__ up, int up_per_row,
                        const float* __restrict__ inverse, float factor,
                        T* __restrict__ grad) {
  __shared__ Sparse sp;
  const float inv_tau = 1.0f / tau;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    T* g = grad + row * classes;
    const int64_t y = labels ? labels[row] : 0;
    const float m = stats[row * 3], s1 = stats[row * 3 + 1];
    const float st = stats[row * 3 + 2];
    if ((labels && y == ignore) || s1 == 0.f) {
      for (int c = threadIdx.x; c < classes; c += kThreads)
        g[c] = narrow<T>(0.f);
      continue;
    }
    const T* z = logits + row * row_stride;
    const float o = origin(m);
    const float scale =
        up[up_per_row ? row : 0] * (inverse ? *inverse : factor);
    const float q_sum =
        load_teacher(sp, values + row * k, index + row * k, k, classes, inv_tau);
    float bad = 0.f;
    float ct = weight == 0.f ? 0.f : weight * tau * q_sum;
    float c1 = 0.f;
    if (labels && weight != 1.f) {
      c1 = 1.f - weight;
      if (!(y >= 0 && y < classes)) bad = __builtin_nanf("");
    }
    const float pt = ct / st * scale + bad, p1 = c1 / s1 * scale;
    for (int c = threadIdx.x; c < classes; c += kThreads) {
      const float d = widen(z[c]) - o;
      g[c] = narrow<T>(pt * exp_of(d * inv_tau) + p1 * exp_of(d));
    }
    __syncthreads();
    // the sparse classes over what the sweep wrote
    for (int j = threadIdx.x; j <= k; j += kThreads) {
      float minus;
      int c;
      if (j < k) {
        bool alone;
        const float q = merged_share(sp, j, k, &alone);
        if (q < 0.f) continue;
        c = sp.column[j];
        minus = weight * tau * q * scale;
        if (c1 != 0.f && c == y) minus += c1 * scale;
      } else {
        if (c1 == 0.f || !(y >= 0 && y < classes)) continue;
        bool seen = false;
        for (int i = 0; i < k; ++i) seen = seen || sp.column[i] == (int)y;
        if (seen) continue;
        c = (int)y;
        minus = c1 * scale;
      }
      const float d = widen(z[c]) - o;
      g[c] = narrow<T>((pt * exp_of(d * inv_tau) + p1 * exp_of(d)) - minus);
    }
    __syncthreads();
  }
}

int grid_of(int64_t rows) { return (int)(rows < 65536 ? rows : 65536); }

}  // namespace

#define ATOMO_BY_TYPE(type, T, ...)                     \
  switch (type) {                                       \
    case ATOMO_F32: { using T = float; __VA_ARGS__; break; }          \
    case ATOMO_BF16: { using T = __hip_bfloat16; __VA_ARGS__; break; } \
    default: { using T = __half; __VA_ARGS__; break; }  \
  }

extern "C" {

void atomo_label_logprobs_launch(const void* logits, int type,
                                 int64_t row_stride, int64_t rows, int classes,
                                 const int64_t* labels, int64_t ignore,
                                 int top, float* logprob, float* entropy,
                                 float* top_logprob, int64_t* top_index,
                                 hipStream_t stream) {
  ATOMO_BY_TYPE(type, T,
                hipLaunchKernelGGL((label_logprobs_kernel<T>), dim3(grid_of(rows)), dim3(kThreads), 0, stream,
                    (const T*)logits, row_stride, rows, classes, labels, ignore,
                    top, logprob, entropy, top_logprob, top_index))
}

void atomo_distill_count_launch(const int64_t* labels, int64_t rows,
                                int64_t ignore, float* inverse,
                                hipStream_t stream) {
  hipLaunchKernelGGL((count_rows_kernel), dim3(1), dim3(1024), 0, stream,
                    labels, rows, ignore, inverse);
}

void atomo_distill_loss_launch(const void* logits, int type, int64_t row_stride,
                               int64_t rows, int classes, const float* values,
                               const int64_t* index, int k,
                               const int64_t* labels, int64_t ignore, float tau,
                               float weight, float* row_loss, float* stats,
                               hipStream_t stream) {
  ATOMO_BY_TYPE(type, T,
                hipLaunchKernelGGL((distill_loss_kernel<T>), dim3(grid_of(rows)), dim3(kThreads), 0, stream,
                    (const T*)logits, row_stride, rows, classes, values, index,
                    k, labels, ignore, tau, weight, row_loss, stats))
}

void atomo_distill_sum_launch(const float* row_loss, int64_t rows,
                              const float* inverse, float factor, float* loss,
                              hipStream_t stream) {
  hipLaunchKernelGGL((sum_rows_kernel), dim3(1), dim3(1024), 0, stream,
                    row_loss, rows, inverse, factor, loss);
}

void atomo_distill_grad_launch(const void* logits, int type, int64_t row_stride,
                               int64_t rows, int classes, const float* values,
                               const int64_t* index, int k,
                               const int64_t* labels, int64_t ignore, float tau,
                               float weight, const float* stats,
                               const float* up, int up_per_row,
                               const float* inverse, float factor, void* grad,
                               hipStream_t stream) {
  ATOMO_BY_TYPE(type, T,
                hipLaunchKernelGGL((distill_grad_kernel<T>), dim3(grid_of(rows)), dim3(kThreads), 0, stream,
                    (const T*)logits, row_stride, rows, classes, values, index,
                    k, labels, ignore, tau, weight, stats, up, up_per_row,
                    inverse, factor, (T*)grad))
}

}  // extern "C"
