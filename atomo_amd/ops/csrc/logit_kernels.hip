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

#include <hip/hip_runtime.h>

#include <cstdint>

#include "logit_kernels.h"

#define WAVE 64

namespace {

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kInf = __builtin_huge_valf();

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
// rows may start at any element: vectors in memory are aligned to elements
typedef u32x4 u32x4_a4 __attribute__((aligned(4)));
typedef u32x4 u32x4_a2 __attribute__((aligned(2)));

__device__ __forceinline__ float nan_value() { return __builtin_nanf(""); }

// -- element types: kVec elements in 16 bytes ---------------------------------
struct F32 {
  using Raw = uint32_t;
  static constexpr int kVec = 4;
  static constexpr Raw kLowest = 0xFF800000u;  // -inf
  using Mem = u32x4_a4;
  __device__ static float widen(Raw r) { return __uint_as_float(r); }
  __device__ static Raw narrow(float f) { return __float_as_uint(f); }
};
struct BF16 {
  using Raw = uint16_t;
  static constexpr int kVec = 8;
  static constexpr Raw kLowest = 0xFF80u;
  using Mem = u32x4_a2;
  __device__ static float widen(Raw r) {
    return __uint_as_float((uint32_t)r << 16);
  }
  __device__ static Raw narrow(float f) {
    return __builtin_bit_cast(Raw, (__bf16)f);
  }
};
struct F16 {
  using Raw = uint16_t;
  static constexpr int kVec = 8;
  static constexpr Raw kLowest = 0xFC00u;
  using Mem = u32x4_a2;
  __device__ static float widen(Raw r) {
    return (float)__builtin_bit_cast(_Float16, r);
  }
  __device__ static Raw narrow(float f) {
    return __builtin_bit_cast(Raw, (_Float16)f);
  }
};

template <typename E>
__device__ __forceinline__ float element(const u32x4& v, int e) {
  if constexpr (E::kVec == 4)
    return E::widen(v[e]);
  else
    return E::widen((uint16_t)(v[e / 2] >> (e % 2 * 16)));
}

// Keeps the compiler from holding the widened elements of `v` over a pass: to
// widen them again costs less than the registers.
__device__ __forceinline__ void forget(u32x4& v) { asm("" : "+v"(v)); }

// 16 bytes from element `at` on; from `end` on, -inf
template <typename E>
__device__ __forceinline__ u32x4 load_vec(const typename E::Raw* z, int at,
                                          int end) {
  if (at + E::kVec <= end) return *(const typename E::Mem*)(z + at);
  u32x4 v;
  if (at >= end) {
    constexpr uint32_t two = E::kLowest | (uint32_t)E::kLowest << 16;
    constexpr uint32_t low = E::kVec == 4 ? (uint32_t)E::kLowest : two;
    return u32x4{low, low, low, low};
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (E::kVec == 4) {
      v[i] = at + i < end ? z[at + i] : E::kLowest;
    } else {
      const uint32_t lo = at + 2 * i < end ? z[at + 2 * i] : E::kLowest;
      const uint32_t hi = at + 2 * i + 1 < end ? z[at + 2 * i + 1] : E::kLowest;
      v[i] = lo | hi << 16;
    }
  }
  return v;
}

template <typename E>
__device__ __forceinline__ void store_vec(typename E::Raw* g, int at, int end,
                                          const float* x) {
  u32x4 v;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (E::kVec == 4)
      v[i] = E::narrow(x[i]);
    else
      v[i] = (uint32_t)E::narrow(x[2 * i]) |
             (uint32_t)E::narrow(x[2 * i + 1]) << 16;
  }
  if (at + E::kVec <= end) {
    *(typename E::Mem*)(g + at) = v;
    return;
  }
#pragma unroll
  for (int e = 0; e < E::kVec; ++e)
    if (at + e < end) g[at + e] = E::narrow(x[e]);
}

// -- sums ---------------------------------------------------------------------
// e^d for d <= 0 (or NaN); e^-inf = 0
__device__ __forceinline__ float exp_of(float d) {
  return __builtin_amdgcn_exp2f(d * kLog2e);
}

// 0 stands in for a maximum of -inf: exp(-inf - 0) is 0, not NaN
__device__ __forceinline__ float origin(float m) { return m == -kInf ? 0.f : m; }

// the exponent that brings a sum relative to `from` to one relative to `to`;
// its floor keeps 0 * -inf out of what it is multiplied with
__device__ __forceinline__ float shift(float from, float to) {
  return fmaxf(from - origin(to), -1e30f);
}

// m, S and T of a part of a row
struct Stat {
  float m, s, t;
  __device__ static Stat none() { return {-kInf, 0.f, 0.f}; }
  __device__ void move(float to) {
    const float d = shift(m, to), f = exp_of(d);
    t = (t + d * s) * f;
    s *= f;
    m = to;
  }
};
// m, S and S_t
struct Sums {
  float m, s, t;
  __device__ static Sums none() { return {-kInf, 0.f, 0.f}; }
  __device__ void move(float to, float inv_tau) {
    const float d = shift(m, to);
    s *= exp_of(d);
    t *= exp_of(d * inv_tau);
    m = to;
  }
};
template <typename P, typename... A>
__device__ __forceinline__ P join(P a, P b, A... tau) {
  const float m = fmaxf(a.m, b.m);
  a.move(m, tau...);
  b.move(m, tau...);
  a.s += b.s;
  a.t += b.t;
  return a;
}

// all lanes get the sum; a fixed order of additions
template <typename P, typename... A>
__device__ __forceinline__ P wave_join(P v, A... tau) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    P o;
    o.m = __shfl_xor(v.m, off, WAVE);
    o.s = __shfl_xor(v.s, off, WAVE);
    o.t = __shfl_xor(v.t, off, WAVE);
    v = (threadIdx.x & off) ? join(o, v, tau...) : join(v, o, tau...);
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

// joins the waves' parts; `lds` holds one for each wave
template <int kThreads, typename P, typename... A>
__device__ __forceinline__ P block_join(P v, P* lds, A... tau) {
  v = wave_join(v, tau...);
  if constexpr (kThreads > WAVE) {
    if (threadIdx.x % WAVE == 0) lds[threadIdx.x / WAVE] = v;
    __syncthreads();
    v = lds[0];
#pragma unroll
    for (int w = 1; w < kThreads / WAVE; ++w) v = join(v, lds[w], tau...);
  }
  return v;
}

// log softmax of one logit
__device__ __forceinline__ float log_prob(float z, float m, float log_s) {
  if (m == -kInf && log_s == -kInf) return -kInf;  // an empty row
  return (z - origin(m)) - log_s;
}

// Rows are spread over two dimensions of the grid: one dimension holds fewer
// than 2^32 threads.
constexpr int kGridRows = 1 << 18;
__device__ __forceinline__ int64_t grid_row(int splits) {
  return (int64_t)blockIdx.y * kGridRows + blockIdx.x / splits;
}
dim3 grid_of(int64_t rows, int splits) {
  const int64_t x = rows < kGridRows ? rows : kGridRows;
  return dim3((unsigned)(x * splits), (unsigned)((rows + x - 1) / x));
}

// -- order of the classes -----------------------------------------------------
// Whole numbers that rise with the value, NaN above all, -0 equal to +0; then
// the lowest class first.  No class has order or key 0.
__device__ __forceinline__ uint32_t order_of(float x) {
  if (x != x) return 0xFFFFFFFFu;
  const uint32_t b = __float_as_uint(x + 0.0f);
  return (b >> 31) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t order) {
  if (order == 0xFFFFFFFFu) return nan_value();
  return __uint_as_float((order >> 31) ? (order & 0x7FFFFFFFu) : ~order);
}
__device__ __forceinline__ uint64_t key_of(float x, int column) {
  return ((uint64_t)order_of(x) << 32) | (0xFFFFFFFFu - (uint32_t)column);
}
__device__ __forceinline__ int column_of(uint64_t key) {
  return (int)(0xFFFFFFFFu - (uint32_t)key);
}

// A wave's candidates for the top k: the classes whose key lies above `bar`.
// The bar never lies above the k-th best key read, and a full list is cut to
// its k best, which raises it.
constexpr int kListSize = 256;

// lanes of one wave read in LDS what others of it wrote
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

__device__ __forceinline__ int count_above(const uint64_t* list, int n,
                                           uint64_t bar) {
  int c = 0;
  for (int i = threadIdx.x % WAVE; i < ((n + WAVE - 1) & -WAVE); i += WAVE)
    c += __popcll(__ballot(i < n && list[i] >= bar));
  return c;
}

// Leaves the k best of n > k distinct keys at the front of the list, in any
// order, and returns a key that exactly they reach.  One wave.
__device__ uint64_t cut_list(uint64_t* list, int n, int k) {
  const int lane = threadIdx.x % WAVE;
  wave_sync();
  // the bits in which the keys differ, from the highest
  uint64_t any = 0, all = ~0ull;
  for (int i = lane; i < n; i += WAVE) {
    any |= list[i];
    all &= list[i];
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    any |= (uint64_t)__shfl_xor((unsigned long long)any, off, WAVE);
    all &= (uint64_t)__shfl_xor((unsigned long long)all, off, WAVE);
  }
  int bit = 63 - __clzll(any ^ all);
  uint64_t bar = bit >= 63 ? 0 : all >> (bit + 1) << (bit + 1);
  int above = n;
  for (; bit >= 0 && above != k; --bit) {
    const uint64_t next = bar | 1ull << bit;
    const int c = count_above(list, n, next);
    if (c >= k) {
      bar = next;
      above = c;
    }
  }
  int kept = 0;
  for (int i = lane; i < ((n + WAVE - 1) & -WAVE); i += WAVE) {
    const uint64_t key = i < n ? list[i] : 0;
    const bool keep = key >= bar && i < n;
    const uint64_t mask = __ballot(keep);
    // written at or before where it was read, and after all lanes' reads
    if (keep) list[kept + __popcll(mask & ((1ull << lane) - 1))] = key;
    kept += __popcll(mask);
  }
  wave_sync();
  return bar;
}

// -- log probabilities --------------------------------------------------------
// One pass over the row makes its sums and leaves, of each thread's chunk of
// kParts loads, the maximum in LDS: 16 bits of its order, cut off downwards.
// The k-th best of the maxima of all loads bounds the k-th best class from
// below, for k classes reach it; so only the few chunks (about k) that reach
// it are read again, out of a cache, and of their classes those that do.
//
// Bound by the memory, and in 16 bits by the vector units: 2048 x 50021 bf16 in
// padded rows with 8 alternatives take 54 us, 3.8 TB/s, at 15.6 vector
// instructions an element, which keep these units busy for 44 us (counted, at
// 2.4 GHz); the memory needs 37.  4096 x 32000 fp32: without alternatives 92 us,
// 5.7 TB/s, with 64 of them 119 us, 4.4 TB/s.  (A large copy reaches 5.5 TB/s.)
// Looking every class up against a bar while it is read took 108 us and 264.
// Rows of equal or rising logits reach any bar everywhere: 512 x 20000 fp32 take
// up to 106 us, else 10.
constexpr int kParts = 4;    // 16-byte loads in flight for each thread
constexpr int kChunks = 16;  // between two selections

// The rank-th best of a wave's maxima, cut to 16 bits.
__device__ __forceinline__ uint32_t wave_bar(const float (&best)[kParts],
                                             int rank) {
  uint32_t order[kParts], low = 0;
#pragma unroll
  for (int u = 0; u < kParts; ++u) order[u] = order_of(best[u]);
  for (int bit = 31; bit >= 16; --bit) {
    const uint32_t c = low | 1u << bit;
    int reach = 0;
#pragma unroll
    for (int u = 0; u < kParts; ++u) reach += __popcll(__ballot(order[u] >= c));
    if (reach >= rank) low = c;
  }
  return low;
}

// One row's results from its sums; one thread.
template <typename E>
__device__ __forceinline__ void write_row(const AtomoLogprobs& a, int64_t row,
                                          const Stat& st, float log_s) {
  a.entropy[row] = st.s == 0.f ? 0.f : log_s - st.t / st.s;
  if (a.labels == nullptr) return;
  const int64_t y = a.labels[row];
  float lp = nan_value();
  if (y == a.ignore)
    lp = 0.f;
  else if (y >= 0 && y < a.classes)
    lp = log_prob(E::widen(((const typename E::Raw*)a.logits)[row * a.row_stride + y]),
                  st.m, log_s);
  a.logprob[row] = lp;
}

// Writes alternative `rank` of a row.
__device__ __forceinline__ void write_top(const AtomoLogprobs& a, int64_t row,
                                          int rank, uint64_t key, float m,
                                          float log_s) {
  a.top_index[row * a.top + rank] = column_of(key);
  a.top_logprob[row * a.top + rank] =
      log_prob(value_of((uint32_t)(key >> 32)), m, log_s);
}

// One workgroup a part of a row.  With one part the row's results are written,
// otherwise the part's sums and its k best keys in order, zeros after them.
template <typename E, int kThreads>
__global__ void __launch_bounds__(kThreads)
    label_logprobs_kernel(AtomoLogprobs a) {
  using Raw = typename E::Raw;
  constexpr int kV = E::kVec, kWaves = kThreads / WAVE;
  constexpr int kChunk = kThreads * kParts * kV;
  constexpr int kOwn = kParts * kV;  // classes of a thread's chunk
  static_assert(kOwn <= WAVE && WAVE % kOwn == 0, "a wave reads whole chunks");
  __shared__ uint64_t lists[kWaves * kListSize];
  __shared__ uint16_t tops[kChunks][kThreads];
  __shared__ uint32_t bars[kWaves];
  __shared__ int counts[kWaves];
  __shared__ Stat stats[kWaves];
  const int64_t row = grid_row(a.splits);
  if (row >= a.rows) return;
  const int part = blockIdx.x % a.splits;
  const int lane = threadIdx.x % WAVE, wave = threadIdx.x / WAVE;
  const Raw* z = (const Raw*)a.logits + row * a.row_stride;
  const int first = part * a.part_size;
  const int end = min(a.classes, first + a.part_size);
  const int top = a.top;
  uint64_t* list = lists + wave * kListSize;
  int n = 0;         // candidates; the same in all lanes of a wave
  uint64_t bar = 0;  // likewise
  float best[kParts];
#pragma unroll
  for (int u = 0; u < kParts; ++u) best[u] = -kInf;
  // Is there a class for each of the first loads of all threads (but for the
  // last part of some rows, always), or, in one wave, for k loads?  Loads
  // without one count as -inf, below no class.
  const bool enough = kWaves > 1 ? end - first >= kThreads * kV
                                 : (end - first + kV - 1) / kV >= top;

  Stat st = Stat::none();
  u32x4 now[kParts], next[kParts];
#pragma unroll
  for (int u = 0; u < kParts; ++u)
    now[u] = load_vec<E>(z, first + (u * kThreads + (int)threadIdx.x) * kV, end);
  for (int s0 = first; s0 < end; s0 += kChunks * kChunk) {
    int chunk = 0;
    for (int c0 = s0; c0 < min(end, s0 + kChunks * kChunk); c0 += kChunk, ++chunk) {
      if (c0 + kChunk < end) {
#pragma unroll
        for (int u = 0; u < kParts; ++u)
          next[u] = load_vec<E>(
              z, c0 + kChunk + (u * kThreads + (int)threadIdx.x) * kV, end);
      }
      float most = -kInf;
#pragma unroll
      for (int u = 0; u < kParts; ++u) {
        float x = element<E>(now[u], 0);
#pragma unroll
        for (int e = 1; e < kV; ++e) x = fmaxf(x, element<E>(now[u], e));
        best[u] = fmaxf(best[u], x);
        most = fmaxf(most, x);
      }
      st.move(fmaxf(st.m, most));
      const float o = origin(st.m);
#pragma unroll
      for (int u = 0; u < kParts; ++u)
#pragma unroll
        for (int e = 0; e < kV; ++e) {
          const float d = element<E>(now[u], e) - o;
          const float x = exp_of(d);
          st.s += x;
          st.t += x * fmaxf(d, -1e30f);
        }
      // NaN is the greatest: once one was summed every chunk is looked at
      if (top > 0)
        tops[chunk][threadIdx.x] =
            st.s != st.s ? 0xFFFF : (uint16_t)(order_of(most) >> 16);
#pragma unroll
      for (int u = 0; u < kParts; ++u) now[u] = next[u];
    }
    if (top == 0) continue;
    // each wave's share of k of the maxima: the least of the bars has k above
    uint32_t low = 0;
    static_assert(ATOMO_LOGIT_TOP_MAX <= WAVE * 4, "a wave's share of k");
    if (enough) low = wave_bar(best, (top + kWaves - 1) / kWaves);
    if (kWaves > 1) {
      __syncthreads();
      if (lane == 0) bars[wave] = low;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < kWaves; ++w) low = min(low, bars[w]);
    }
    if (low != 0) {
      const uint64_t at_least = ((uint64_t)low << 32) - 1;
      bar = at_least > bar ? at_least : bar;
    }
    wave_sync();
    for (int c = 0; c < chunk; ++c) {
      uint64_t hits = __ballot(tops[c][threadIdx.x] >= (uint32_t)((bar + 1) >> 48));
      while (hits != 0) {
        // the next chunks that reach the bar, a lane for each of their classes
        int who = -1;
#pragma unroll
        for (int g = 0; g < WAVE / kOwn; ++g) {
          const int bit = hits ? __builtin_ctzll(hits) : -1;
          if (lane / kOwn == g) who = bit;
          hits &= hits - 1;
        }
        const int own = lane % kOwn;
        const int at = s0 + c * kChunk +
                       (own / kV * kThreads + wave * WAVE + who) * kV + own % kV;
        const bool there = who >= 0 && at < end;
        const uint64_t key = there ? key_of(E::widen(z[at]), at) : 0;
        uint64_t mask = __ballot(key > bar);
        if (n + __popcll(mask) > kListSize) {
          bar = cut_list(list, n, top) - 1;
          n = top;
          mask = __ballot(key > bar);
        }
        if (key > bar) list[n + __popcll(mask & ((1ull << lane) - 1))] = key;
        n += __popcll(mask);
      }
    }
    if (kWaves > 1) __syncthreads();  // `bars` is written again
  }

  st = block_join<kThreads>(st, stats);
  const float log_s = logf(st.s);
  if (top > 0) {
    if (lane == 0) counts[wave] = n;
    __syncthreads();
    // A key's rank is the number of greater ones: of n candidates, mostly a
    // little over k, n^2 / 256 reads for each thread.
    int all = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) all += counts[w];
    for (int i = threadIdx.x; i < all; i += kThreads) {
      int w = 0, j = i;
      while (j >= counts[w]) j -= counts[w++];
      const uint64_t key = lists[w * kListSize + j];
      int rank = 0;
      for (w = 0; w < kWaves; ++w)
        for (j = 0; j < counts[w]; ++j) rank += lists[w * kListSize + j] > key;
      if (rank >= top) continue;
      if (a.splits > 1)
        a.part_keys[(row * a.splits + part) * top + rank] = (int64_t)key;
      else
        write_top(a, row, rank, key, st.m, log_s);
    }
    if (a.splits > 1)
      for (int i = all + threadIdx.x; i < top; i += kThreads)
        a.part_keys[(row * a.splits + part) * top + i] = 0;
  }
  if (threadIdx.x == 0) {
    if (a.splits > 1) {
      float* p = a.part_stat + (row * a.splits + part) * 3;
      p[0] = st.m;
      p[1] = st.s;
      p[2] = st.t;
    } else {
      write_row<E>(a, row, st, log_s);
    }
  }
}

// Joins a row's parts: one workgroup a row.  A part's last key, where it has
// k, is a bar for all of them; so is the least of the parts' d-th keys, where
// d keys of each are k together, and mostly the higher one.  Bound by latency:
// one row of 131072 bf16 with 20 alternatives takes 10 us in 16 parts and 5 us
// here, 22 us in all with 128.
constexpr int kMostSplits = ATOMO_LOGIT_MAX_SPLITS;
constexpr int kJoin = 256;

template <typename E>
__global__ void __launch_bounds__(kJoin)
    join_logprobs_kernel(AtomoLogprobs a) {
  __shared__ uint64_t list[kMostSplits * ATOMO_LOGIT_TOP_MAX];
  __shared__ int count;
  static_assert(kMostSplits <= WAVE, "a lane joins one part");
  const int64_t row = grid_row(1);
  if (row >= a.rows) return;
  const int lane = threadIdx.x % WAVE, top = a.top;
  const uint64_t* keys = (const uint64_t*)a.part_keys + row * a.splits * top;
  Stat st = Stat::none();
  const int share = (top + a.splits - 1) / a.splits;
  uint64_t bar = 1, least = ~0ull;
  if (lane < a.splits) {
    const float* p = a.part_stat + (row * a.splits + lane) * 3;
    st = {p[0], p[1], p[2]};
    if (top > 0) {
      bar = max(bar, keys[lane * top + top - 1]);
      least = keys[lane * top + share - 1];
    }
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    bar = max(bar, (uint64_t)__shfl_xor((unsigned long long)bar, off, WAVE));
    least = min(least, (uint64_t)__shfl_xor((unsigned long long)least, off, WAVE));
  }
  bar = max(bar, least);
  st = wave_join(st);
  const float log_s = logf(st.s);
  if (threadIdx.x == 0) {
    count = 0;
    write_row<E>(a, row, st, log_s);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < a.splits * top; i += kJoin) {
    const uint64_t key = keys[i];
    if (key >= bar) list[atomicAdd(&count, 1)] = key;
  }
  __syncthreads();
  // keys are distinct: their order in the list does not matter
  const int n = count;
  for (int i = threadIdx.x; i < n; i += kJoin) {
    const uint64_t key = list[i];
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += list[j] > key;
    if (rank < top) write_top(a, row, rank, key, st.m, log_s);
  }
}

// -- distillation -------------------------------------------------------------
using Distill = AtomoDistill;

// What exp(d) costs beside exp(d / tau): nothing at tau 1, a square at 2, two
// at 4 (each a rounding of half a step), an exponential of its own elsewhere.
// Training on 4096 x 65536 bf16 / 4096 x 32000 fp32 / 1001 x 50021 fp16, tau 2:
// 234 / 215 / 81 us, tau 3: 243 / 216 / 84; the loss alone 111 / 103 / 37 and
// 117 / 106 / 40.
enum Mode {
  kSoftOnly = ATOMO_DISTILL_SOFT,
  kTau1 = ATOMO_DISTILL_TAU1,
  kTau2 = ATOMO_DISTILL_TAU2,
  kTau4 = ATOMO_DISTILL_TAU4
};

__device__ __forceinline__ float hard_exp(int mode, float d, float soft) {
  if (mode == kTau1) return soft;
  if (mode == kTau2) return soft * soft;
  if (mode == kTau4) {
    const float s = soft * soft;
    return s * s;
  }
  return exp_of(d);
}

// A teacher's row and the label in the registers of the first wave: a lane
// holds entries lane and lane + 64.
struct Teacher {
  int64_t at[2];     // as given
  int column[2];     // -1: absent, or an earlier entry stands for its class
  float q[2], lq[2]; // of the class: q and its logarithm (first, the value)
  float z[2];        // the student's logit there
  float sum;         // of q: 1, 0 for no entry, NaN for a wrong one
  bool hard;         // a label counts
  float zy;          // the student's logit at the label, NaN for a wrong one
  int y;             // the label, -1 for a wrong one
  bool seen;         // the label is among the entries

  // Reads a row's entries, all lanes of the first wave; nothing waits for them.
  __device__ void fetch(const Distill& a, int64_t row) {
    const int lane = threadIdx.x % WAVE;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int j = lane + h * WAVE;
      lq[h] = j < a.k ? a.values[row * a.k + j] : -kInf;
      at[h] = j < a.k ? a.index[row * a.k + j] : -1;
    }
  }

  template <typename E>
  __device__ void read(const Distill& a, const typename E::Raw* z_row,
                       int64_t label) {
    const int lane = threadIdx.x % WAVE;
    bool wrong = false;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const bool there = lq[h] != -kInf, in = at[h] >= 0 && at[h] < a.classes;
      wrong |= there && !in;
      column[h] = there && in ? (int)at[h] : -1;
      // used with the sums only, long after
      z[h] = column[h] < 0 ? 0.f : E::widen(z_row[column[h]]);
    }
    hard = a.labels != nullptr && a.rest != 0.f;
    y = -1;
    zy = nan_value();
    if (hard && label >= 0 && label < a.classes) {
      y = (int)label;
      zy = E::widen(z_row[label]);
    }
    const float o = origin(wave_max(fmaxf(lq[0], lq[1])));
    const float s = wave_sum(exp_of((lq[0] - o) * a.inv_tau) +
                             exp_of((lq[1] - o) * a.inv_tau));
    const float log_s = logf(s);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      lq[h] = column[h] < 0 ? -kInf : (lq[h] - o) * a.inv_tau - log_s;
      q[h] = column[h] < 0 ? 0.f : exp_of(lq[h]);
    }
    sum = s == 0.f ? 0.f : (s == s ? 1.f : s);
    if (__ballot(wrong) != 0) sum = nan_value();
    // is a class there twice?
    bool twice = false;
    for (int d = 1; d <= WAVE / 2; ++d)
      twice |= column[0] >= 0 &&
               column[0] == __shfl(column[0], (lane + d) % WAVE, WAVE);
    if (a.k > WAVE)
      for (int d = 0; d < WAVE; ++d) {
        const int c = __shfl(column[1], (lane + d) % WAVE, WAVE);
        twice |= c >= 0 && (c == column[0] || (d > 0 && c == column[1]));
      }
    if (__ballot(twice) != 0) merge(a);
    seen = __ballot(y >= 0 && (column[0] == y || column[1] == y)) != 0;
  }

  // entries of one class: the first stands for all
  __device__ void merge(const Distill& a) {
    const int lane = threadIdx.x % WAVE;
    bool later[2] = {false, false};
    float more[2] = {0.f, 0.f};
    for (int j = 0; j < a.k; ++j) {
      const int h = j / WAVE;
      const int c = __builtin_amdgcn_readlane(h ? column[1] : column[0], j % WAVE);
      const float qj = __uint_as_float(__builtin_amdgcn_readlane(
          __float_as_uint(h ? q[1] : q[0]), j % WAVE));
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        if (column[g] != c || lane + g * WAVE == j) continue;
        later[g] |= j < lane + g * WAVE;
        more[g] += qj;
      }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (column[h] >= 0 && !later[h] && more[h] > 0.f) {
        q[h] += more[h];
        lq[h] = logf(q[h]);
      }
      if (later[h]) column[h] = -1;
    }
  }

  // the row's loss; all lanes of the first wave
  __device__ float loss(const Distill& a, const Sums& st) const {
    if (st.s == 0.f) return 0.f;  // a row of -inf only
    const float o = origin(st.m), log_st = logf(st.t);
    float kd = 0.f;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (column[h] < 0) continue;
      if (!(q[h] <= 0.f))
        kd += q[h] * (lq[h] - ((z[h] - o) * a.inv_tau - log_st));
    }
    kd = wave_sum(kd);
    float row = 0.f;
    if (a.k != 0)
      row = a.weight * a.tau * a.tau * (sum != sum ? sum : kd);
    if (hard) row += a.rest * (logf(st.s) - (zy - o));
    return row;
  }

  // dz of the entries' classes and the label's within [first, end), over what
  // the sweep wrote there; ct and c1 as in Factors
  template <typename E>
  __device__ void patch(const Distill& a, const Sums& st, float pt, float p1,
                        float ct, float c1, typename E::Raw* g, int first,
                        int end) const {
    const float o = origin(st.m);
    const auto put = [&](int c, float zc, float minus) {
      if (c < first || c >= end) return;
      const float d = zc - o;
      const float soft = exp_of(d * a.inv_tau);
      float x = pt * soft;
      if (a.mode != kSoftOnly) x += p1 * hard_exp(a.mode, d, soft);
      g[c] = E::narrow(x - minus);
    };
#pragma unroll
    for (int h = 0; h < 2; ++h)
      if (column[h] >= 0)
        put(column[h], z[h], ct * q[h] + (hard && column[h] == y ? c1 : 0.f));
    if (hard && y >= 0 && !seen && threadIdx.x % WAVE == 0) put(y, zy, c1);
  }
};

// Rows that a mean counts: all lanes of the first wave.
__device__ __forceinline__ float inverse_count(const Distill& a) {
  if (a.inverse != nullptr) return *a.inverse;
  if (!a.count) return a.factor;
  int n = 0;
  for (int64_t i = threadIdx.x % WAVE; i < a.rows; i += WAVE)
    n += a.labels[i] != a.ignore;
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) n += __shfl_xor(n, off, WAVE);
  return 1.0f / (float)(n > 0 ? n : 1);
}

template <typename E>
__device__ __forceinline__ void add_exps(const u32x4& v, float o, float inv_tau,
                                         int mode, Sums& st) {
  float soft[E::kVec];
  const float c = inv_tau * kLog2e;
#pragma unroll
  for (int e = 0; e < E::kVec; ++e) {
    soft[e] = __builtin_amdgcn_exp2f((element<E>(v, e) - o) * c);
    st.t += soft[e];
  }
  if (mode == kSoftOnly) return;
  if (mode == kTau1) {
#pragma unroll
    for (int e = 0; e < E::kVec; ++e) st.s += soft[e];
  } else if (mode == kTau2) {
#pragma unroll
    for (int e = 0; e < E::kVec; ++e) st.s += soft[e] * soft[e];
  } else if (mode == kTau4) {
#pragma unroll
    for (int e = 0; e < E::kVec; ++e) {
      const float s = soft[e] * soft[e];
      st.s += s * s;
    }
  } else {
#pragma unroll
    for (int e = 0; e < E::kVec; ++e) st.s += exp_of(element<E>(v, e) - o);
  }
}

template <typename E>
__device__ __forceinline__ void write_grad(const u32x4& v, float o,
                                           float inv_tau, int mode, float pt,
                                           float p1, typename E::Raw* g, int at,
                                           int end) {
  if (at >= end) return;
  float x[E::kVec];
  const float c = inv_tau * kLog2e;
#pragma unroll
  for (int e = 0; e < E::kVec; ++e)
    x[e] = __builtin_amdgcn_exp2f((element<E>(v, e) - o) * c);
  if (mode == kSoftOnly) {
#pragma unroll
    for (int e = 0; e < E::kVec; ++e) x[e] *= pt;
  } else if (mode == kTau1) {
    const float p = pt + p1;
#pragma unroll
    for (int e = 0; e < E::kVec; ++e) x[e] *= p;
  } else if (mode == kTau2) {
#pragma unroll
    for (int e = 0; e < E::kVec; ++e) x[e] = x[e] * (pt + p1 * x[e]);
  } else if (mode == kTau4) {
#pragma unroll
    for (int e = 0; e < E::kVec; ++e) {
      const float s = x[e] * x[e];
      x[e] = pt * x[e] + p1 * (s * s);
    }
  } else {
#pragma unroll
    for (int e = 0; e < E::kVec; ++e)
      x[e] = pt * x[e] + p1 * exp_of(element<E>(v, e) - o);
  }
  store_vec<E>(g, at, end, x);
}

template <typename E, int kThreads>
__device__ __forceinline__ void write_zeros(typename E::Raw* g, int first,
                                            int end) {
  const float zero[E::kVec] = {};
  for (int at = first + (int)threadIdx.x * E::kVec; at < end;
       at += kThreads * E::kVec)
    store_vec<E>(g, at, end, zero);
}

// Loss and, where it is wanted, gradient of a row that fits a workgroup's
// registers, kLoads 16-byte loads a thread: the logits are read once.  Bound by
// the memory: 4096 x 65536 bf16 with an eighth of the rows ignored in 223 us,
// 4.5 TB/s.  Four waves a SIMD, that is two workgroups of 512 a CU, matter: one
// reads while the other sums (190 registers, one workgroup: 351 us).  Reading
// the next row ahead into registers instead spilled, 400 us.
template <typename E, int kThreads, int kLoads>
__global__ void __launch_bounds__(kThreads)
    __attribute__((amdgpu_waves_per_eu(4))) distill_fused_kernel(Distill a) {
  constexpr int kV = E::kVec, kWaves = kThreads / WAVE;
  __shared__ float lds_max[kWaves];
  __shared__ Sums lds_sums[kWaves];
  __shared__ float lds_scale, lds_sum;
  const int64_t row = grid_row(1);
  if (row >= a.rows) return;
  using Raw = typename E::Raw;
  const Raw* z = (const Raw*)a.logits + row * a.row_stride;
  Raw* g = (Raw*)a.grad + row * a.classes;
  const int64_t label = a.labels ? a.labels[row] : 0;
  if (a.labels && label == a.ignore) {
    if (a.grad) write_zeros<E, kThreads>(g, 0, a.classes);
    if (threadIdx.x == 0) a.row_loss[row] = 0.f;
    return;
  }
  u32x4 v[kLoads];
#pragma unroll
  for (int r = 0; r < kLoads; ++r)
    v[r] = load_vec<E>(z, (r * kThreads + (int)threadIdx.x) * kV, a.classes);
  const int wave = threadIdx.x / WAVE;
  Teacher teacher;
  if (wave == 0) {
    teacher.fetch(a, row);
    teacher.read<E>(a, z, label);
    const float scale = inverse_count(a);
    if (threadIdx.x == 0) {
      lds_scale = scale;
      lds_sum = teacher.sum;
    }
  }
  float m = -kInf;
#pragma unroll
  for (int r = 0; r < kLoads; ++r)
#pragma unroll
    for (int e = 0; e < kV; ++e) m = fmaxf(m, element<E>(v[r], e));
  m = wave_max(m);
  if (threadIdx.x % WAVE == 0) lds_max[wave] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) m = fmaxf(m, lds_max[w]);
  const float o = origin(m);
  Sums st = {m, 0.f, 0.f};
#pragma unroll
  for (int r = 0; r < kLoads; ++r) {
    forget(v[r]);
    if (r * kThreads * kV < a.classes)
      add_exps<E>(v[r], o, a.inv_tau, a.mode, st);
  }
  st.s = wave_sum(st.s);
  st.t = wave_sum(st.t);
  if (threadIdx.x % WAVE == 0) lds_sums[wave] = st;
  __syncthreads();
  st.s = st.t = 0.f;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    st.s += lds_sums[w].s;
    st.t += lds_sums[w].t;
  }
  if (a.mode == kSoftOnly) st.s = st.t;  // only whether it is 0 is asked
  const float scale = lds_scale, q_sum = lds_sum;
  const bool hard = a.labels != nullptr && a.rest != 0.f;
  const float ct = a.k == 0 ? 0.f : a.weight * a.tau * scale;
  float c1 = hard ? a.rest * scale : 0.f;
  const float wrong =
      hard && !(label >= 0 && label < a.classes) ? nan_value() : 0.f;
  if (wave == 0) {
    const float loss = teacher.loss(a, st);
    if (threadIdx.x == 0) {
      a.row_loss[row] = loss;
      float* p = a.stats + row * a.splits * 3;
      p[0] = st.m;
      p[1] = st.s;
      p[2] = st.t;
    }
  }
  if (a.grad == nullptr) return;
  // no distribution, or no term at all: a teacher without an entry adds nothing
  // to the gradient of a NaN, either
  if (st.s == 0.f || (!hard && q_sum == 0.f)) {
    write_zeros<E, kThreads>(g, 0, a.classes);
    return;
  }
  const float pt = (a.k == 0 ? 0.f : ct * q_sum) / st.t + wrong;
  const float p1 = c1 / st.s;
#pragma unroll
  for (int r = 0; r < kLoads; ++r) {
    forget(v[r]);
    write_grad<E>(v[r], o, a.inv_tau, a.mode, pt, p1, g,
                  (r * kThreads + (int)threadIdx.x) * kV, a.classes);
  }
  __syncthreads();
  if (wave == 0) teacher.patch<E>(a, st, pt, p1, ct, c1, g, 0, a.classes);
}

constexpr int kSweep = 256;

// The sums of a part of a row, and of a whole one the loss: a sweep with the
// running maximum.  Bound by the memory: 4096 x 32000 fp32 with an eighth of
// the rows ignored in 89 us, 5.2 TB/s; 1001 x 50021 fp16 in 28 us, 3.6 TB/s.
template <typename E>
__global__ void __launch_bounds__(kSweep) distill_sums_kernel(Distill a) {
  constexpr int kV = E::kVec;
  constexpr int kChunk = kSweep * kParts * kV;
  __shared__ Sums lds[kSweep / WAVE];
  const int64_t row = grid_row(a.splits);
  if (row >= a.rows) return;
  const int part = blockIdx.x % a.splits;
  const int64_t label = a.labels ? a.labels[row] : 0;
  if (a.labels && label == a.ignore) {
    if (a.splits == 1 && threadIdx.x == 0) a.row_loss[row] = 0.f;
    return;
  }
  const typename E::Raw* z =
      (const typename E::Raw*)a.logits + row * a.row_stride;
  const int first = part * a.part_size;
  const int end = min(a.classes, first + a.part_size);
  Sums st = Sums::none();
  u32x4 now[kParts], next[kParts];
#pragma unroll
  for (int u = 0; u < kParts; ++u)
    now[u] = load_vec<E>(z, first + (u * kSweep + (int)threadIdx.x) * kV, end);
  for (int c0 = first; c0 < end; c0 += kChunk) {
    if (c0 + kChunk < end) {
#pragma unroll
      for (int u = 0; u < kParts; ++u)
        next[u] = load_vec<E>(
            z, c0 + kChunk + (u * kSweep + (int)threadIdx.x) * kV, end);
    }
    float m = st.m;
#pragma unroll
    for (int u = 0; u < kParts; ++u)
#pragma unroll
      for (int e = 0; e < kV; ++e) m = fmaxf(m, element<E>(now[u], e));
    st.move(m, a.inv_tau);
    const float o = origin(m);
#pragma unroll
    for (int u = 0; u < kParts; ++u)
      add_exps<E>(now[u], o, a.inv_tau, a.mode, st);
#pragma unroll
    for (int u = 0; u < kParts; ++u) now[u] = next[u];
  }
  st = block_join<kSweep>(st, lds, a.inv_tau);
  if (a.mode == kSoftOnly) st.s = st.t;
  if (threadIdx.x == 0) {
    float* p = a.stats + (row * a.splits + part) * 3;
    p[0] = st.m;
    p[1] = st.s;
    p[2] = st.t;
  }
  if (a.splits == 1 && threadIdx.x < WAVE) {
    Teacher teacher;
    teacher.fetch(a, row);
    teacher.read<E>(a, z, label);
    const float loss = teacher.loss(a, st);
    if (threadIdx.x == 0) a.row_loss[row] = loss;
  }
}

__device__ __forceinline__ Sums row_sums(const Distill& a, int64_t row) {
  Sums st = Sums::none();
  const int lane = threadIdx.x % WAVE;
  if (lane < a.splits) {
    const float* p = a.stats + (row * a.splits + lane) * 3;
    st = {p[0], p[1], p[2]};
  }
  return wave_join(st, a.inv_tau);
}

// The split rows' losses from their sums: one wave a row, bound by latency.
template <typename E>
__global__ void __launch_bounds__(WAVE) distill_loss_kernel(Distill a) {
  const int64_t row = grid_row(1);
  if (row >= a.rows) return;
  const int64_t label = a.labels ? a.labels[row] : 0;
  float loss = 0.f;
  if (!(a.labels && label == a.ignore)) {
    Teacher teacher;
    teacher.fetch(a, row);
    teacher.read<E>(a, (const typename E::Raw*)a.logits + row * a.row_stride,
                    label);
    loss = teacher.loss(a, row_sums(a, row));
  }
  if (threadIdx.x == 0) a.row_loss[row] = loss;
}

// The gradient of a part of a row from the row's sums.  Bound by the memory:
// 1001 x 50021 fp16 in 41 us, 4.9 TB/s.
template <typename E>
__global__ void __launch_bounds__(kSweep) distill_grad_kernel(Distill a) {
  constexpr int kV = E::kVec;
  __shared__ float lds_scale, lds_sum;
  // the forward pass wrote the gradient for an upstream one of 1
  if (a.skip_one && *a.up == 1.f) return;
  const int64_t row = grid_row(a.grad_splits);
  if (row >= a.rows) return;
  const int part = blockIdx.x % a.grad_splits;
  using Raw = typename E::Raw;
  const Raw* z = (const Raw*)a.logits + row * a.row_stride;
  Raw* g = (Raw*)a.grad + row * a.classes;
  const int first = part * a.grad_part;
  const int end = min(a.classes, first + a.grad_part);
  const int64_t label = a.labels ? a.labels[row] : 0;
  if (a.labels && label == a.ignore) {
    write_zeros<E, kSweep>(g, first, end);
    return;
  }
  const Sums st = row_sums(a, row);
  if (st.s == 0.f) {
    write_zeros<E, kSweep>(g, first, end);
    return;
  }
  const int wave = threadIdx.x / WAVE;
  Teacher teacher;
  if (wave == 0) {
    teacher.fetch(a, row);
    teacher.read<E>(a, z, label);
    const float scale = inverse_count(a) * a.up[a.up_per_row ? row : 0];
    if (threadIdx.x == 0) {
      lds_scale = scale;
      lds_sum = teacher.sum;
    }
  }
  __syncthreads();
  const float scale = lds_scale, q_sum = lds_sum;
  const float o = origin(st.m);
  const bool hard = a.labels != nullptr && a.rest != 0.f;
  const float ct = a.k == 0 ? 0.f : a.weight * a.tau * scale;
  const float c1 = hard ? a.rest * scale : 0.f;
  const float wrong =
      hard && !(label >= 0 && label < a.classes) ? nan_value() : 0.f;
  if (!hard && q_sum == 0.f) {  // no term at all, whatever the logits are
    write_zeros<E, kSweep>(g, first, end);
    return;
  }
  const float pt = (a.k == 0 ? 0.f : ct * q_sum) / st.t + wrong;
  const float p1 = c1 / st.s;
  for (int c0 = first; c0 < end; c0 += kSweep * kParts * kV) {
    u32x4 v[kParts];
#pragma unroll
    for (int u = 0; u < kParts; ++u)
      v[u] = load_vec<E>(z, c0 + (u * kSweep + (int)threadIdx.x) * kV, end);
#pragma unroll
    for (int u = 0; u < kParts; ++u)
      write_grad<E>(v[u], o, a.inv_tau, a.mode, pt, p1, g,
                    c0 + (u * kSweep + (int)threadIdx.x) * kV, end);
  }
  __syncthreads();
  if (wave == 0) teacher.patch<E>(a, st, pt, p1, ct, c1, g, first, end);
}

// Rows that count, and the rows' losses added up in a fixed order: one
// workgroup, bound by latency (4096 rows: 3 and 5 us).
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
    int64_t all = 0;
    for (int i = 0; i < 1024 / WAVE; ++i) all += lds[i];
    *inverse = 1.0f / (float)(all > 0 ? all : 1);
  }
}

__global__ void __launch_bounds__(1024)
    sum_rows_kernel(Distill a, float* __restrict__ loss) {
  __shared__ float lds[1024 / WAVE];
  // scaled before they are added: a mean of huge rows stays finite
  const float each = inverse_count(a);
  float v = 0.f;
  for (int64_t i = threadIdx.x; i < a.rows; i += 1024) v += a.row_loss[i] * each;
  v = wave_sum(v);
  if (threadIdx.x % WAVE == 0) lds[threadIdx.x / WAVE] = v;
  __syncthreads();
  if (threadIdx.x == 0) {
    float all = 0.f;
    for (int i = 0; i < 1024 / WAVE; ++i) all += lds[i];
    *loss = all;
  }
}

// A row is split where there are too few rows to fill the card, evenly, and so
// that the parts are not much below a chunk of a 256-thread workgroup.
constexpr int kFill = 512;  // workgroups: two for each of 256 CUs

int splits_of(int64_t rows, int classes, int vec, int* part) {
  if (rows < 1) rows = 1;
  const int64_t chunk = 256 * kParts * vec;
  int64_t n = (kFill + rows - 1) / rows;
  n = n < kMostSplits ? n : kMostSplits;
  const int64_t chunks = (classes + chunk - 1) / chunk;
  n = n < chunks ? n : chunks;
  if (n <= 1) {
    *part = classes;
    return 1;
  }
  const int64_t size = ((classes + n - 1) / n + vec - 1) / vec * vec;
  *part = (int)size;
  return (int)((classes + size - 1) / size);
}

int vec_of(int type) { return type == ATOMO_F32 ? 4 : 8; }

template <typename E>
void label_logprobs(const AtomoLogprobs& a, hipStream_t stream) {
  // one wave for a row that it holds in one chunk
  if (a.splits == 1 && a.classes <= WAVE * kParts * E::kVec) {
    hipLaunchKernelGGL((label_logprobs_kernel<E, WAVE>), grid_of(a.rows, 1),
                       dim3(WAVE), 0, stream, a);
    return;
  }
  hipLaunchKernelGGL((label_logprobs_kernel<E, 256>), grid_of(a.rows, a.splits),
                     dim3(256), 0, stream, a);
  if (a.splits > 1)
    hipLaunchKernelGGL((join_logprobs_kernel<E>), grid_of(a.rows, 1),
                       dim3(kJoin), 0, stream, a);
}

template <typename E, int kThreads, int kLoads>
void launch_fused(const Distill& a, hipStream_t stream) {
  hipLaunchKernelGGL((distill_fused_kernel<E, kThreads, kLoads>), grid_of(a.rows, 1),
                     dim3(kThreads), 0, stream, a);
}

// The smallest workgroup whose registers hold a row: more of them share a CU,
// and one's loads run beside another's sums.
template <typename E>
void distill_fused(const Distill& a, hipStream_t stream) {
  const int loads = (a.classes + E::kVec - 1) / E::kVec;
  if (loads <= 64)
    launch_fused<E, 64, 1>(a, stream);
  else if (loads <= 64 * 4)
    launch_fused<E, 64, 4>(a, stream);
  else if (loads <= 64 * 16)
    launch_fused<E, 64, 16>(a, stream);
  else if (loads <= 256 * 16)
    launch_fused<E, 256, 16>(a, stream);
  else if (loads <= 512 * 16)
    launch_fused<E, 512, 16>(a, stream);
  else
    launch_fused<E, 1024, 16>(a, stream);
}

template <typename E>
void distill_loss(const Distill& a, hipStream_t stream) {
  hipLaunchKernelGGL((distill_sums_kernel<E>), grid_of(a.rows, a.splits),
                     dim3(kSweep), 0, stream, a);
  if (a.splits == 1) return;
  hipLaunchKernelGGL((distill_loss_kernel<E>), grid_of(a.rows, 1), dim3(WAVE), 0,
                     stream, a);
}

template <typename E>
void distill_grad(const Distill& a, hipStream_t stream) {
  hipLaunchKernelGGL((distill_grad_kernel<E>), grid_of(a.rows, a.grad_splits),
                     dim3(kSweep), 0, stream, a);
}

}  // namespace

#define ATOMO_BY_TYPE(type, call)      \
  switch (type) {                      \
    case ATOMO_F32: call<F32>(*a, stream); break;   \
    case ATOMO_BF16: call<BF16>(*a, stream); break; \
    default: call<F16>(*a, stream);    \
  }

extern "C" {

int atomo_logit_splits(int64_t rows, int classes, int type, int* part_size) {
  return splits_of(rows, classes, vec_of(type), part_size);
}

void atomo_label_logprobs_launch(const AtomoLogprobs* a, hipStream_t stream) {
  ATOMO_BY_TYPE(a->type, label_logprobs)
}

int atomo_distill_short(int classes, int type) {
  return classes <= WAVE * 16 * vec_of(type);
}

int atomo_distill_fits(int64_t rows, int classes, int type) {
  // of fewer rows each is split, so as to fill the card
  return atomo_distill_short(classes, type) ||
         (classes <= 1024 * 16 * vec_of(type) && rows >= 128);
}

void atomo_distill_count_launch(const int64_t* labels, int64_t rows,
                                int64_t ignore, float* inverse,
                                hipStream_t stream) {
  hipLaunchKernelGGL(count_rows_kernel, dim3(1), dim3(1024), 0, stream, labels,
                     rows, ignore, inverse);
}

void atomo_distill_fused_launch(const AtomoDistill* a, hipStream_t stream) {
  ATOMO_BY_TYPE(a->type, distill_fused)
}

void atomo_distill_loss_launch(const AtomoDistill* a, hipStream_t stream) {
  ATOMO_BY_TYPE(a->type, distill_loss)
}

void atomo_distill_sum_launch(const AtomoDistill* a, float* loss,
                              hipStream_t stream) {
  hipLaunchKernelGGL(sum_rows_kernel, dim3(1), dim3(1024), 0, stream, *a, loss);
}

void atomo_distill_grad_launch(const AtomoDistill* a, hipStream_t stream) {
  ATOMO_BY_TYPE(a->type, distill_grad)
}

}  // extern "C"
